// Dense products of the feed-forward layers on the tcgen05 tensor cores: 8-bit
// products with row and channel scales, the gated block's forward pass and its
// gradients.
//
// One persistent kernel. A CTA pair computes a tile of 256 rows x 256 accumulator
// columns; each CTA stages its 128 rows of A and its 128 rows of B (half the
// tile's columns) per K block of 128 bytes, six blocks deep, with TMA into
// 128-byte-swizzled tiles. Against one CTA per 128 x 256 tile this reads a third
// less from L2 per product, which is what bounds a tile loop at this size.
// Warp 0 loads, warp 1 of the leader issues the MMAs, warps 2-17 read the
// accumulators (TMEM lane = row) and write the results; two accumulator buffers of
// 256 columns, so that a tile's epilogue runs under the next tile's MMAs.
//
// Operands are K-major (the contraction runs along the row) or MN-major (it runs
// down the rows): the gradients need transposed operands, and the tensor core
// reads them in place. An operand whose rows do not start on 16-byte boundaries
// (TMA's rule) is first copied into padded rows.
//
// Tiles beyond the last whole wave (one tile a CTA pair) of a long contraction are
// split along K, so that they fill the pairs too: each part writes raw 32-bit sums,
// k_join adds them in order.
//
// Sums are float32 (int32 for 8-bit operands). What goes from one product to the next is
// rounded to the element type, because the tensor core takes 16-bit operands: h = silu(g) u
// in the forward pass, dg and du in the gradient, each from float32 accumulators and
// rounded once. Two independent roundings instead of one: a training step's results are
// 1.4 times as far from 64-bit ones as a float32 chain's that is rounded at its end (2-norm:
// bfloat16 0.0023 and 0.0017 at 24000 x 256 x 1024, float16 0.00029 and 0.00021 at 8190 x
// 2048 x 8200). Keeping h, dg and du in two parts would add two thirds
// to the products.
//
// Every wait is bounded (layers.hpp, WaitLimit) and waits for one step of the pipeline.
// After one that gives up, the pair ends what it has started before it leaves.
#include <atomic>
#include <cstring>
#include <string>

#include "layers_common.cuh"
#include "model_host.hpp"
#include "tensor_core.cuh"

namespace so3lr_b200 {
namespace {

constexpr int kPairs = kSmCount / 2;
constexpr int kTileM = 256;                 // rows of a CTA pair's tile
constexpr int kEpiWarps = 16;  // four a scheduler: with two the epilogue's latencies show
constexpr int kThreads = (2 + kEpiWarps) * 32;
constexpr uint32_t kOperand = 128 * 128;    // 128 rows of 128 bytes: one operand tile of a CTA, 16 KB
constexpr uint32_t kStaging = 2048;         // of an epilogue warp: 32 rows x 64 bytes
constexpr int kBarBytes = 256;
constexpr int kMaxMaps = 6, kMaxProblems = 3, kMaxStages = 8;
constexpr int kItemTable = 32;              // work items of a pair worked out once, at its start

// What the kernel computes.
enum Mode {
  kPlain,     // C = A B^T, one or two K segments (A1 B1^T + A2 B2^T)
  kInt8,      // C = (A B^T) a_scale b_scale + bias
  kGated,     // C = silu(A G^T) * (A U^T): 128 columns of G and 128 of U per tile
  kGatedBack, // g, u as above and dh = DY Wd: C = dg, C2 = du
  kKeptBack   // the same with g, u read from the forward pass: dh alone is computed
};
// Accumulator columns of a tile, TN: 256, or 128 where 256 would leave most pairs
// without a tile. A narrow tile takes half the time a K block, and there are twice as
// many; it reads half as much again from L2 for each product.
template <int MODE, int TN>
struct Shape {
  static constexpr uint32_t kOperandB = TN * 64;  // TN / 2 rows of 128 bytes
  // x, dy, one of Wg / Wu, 64 columns of Wd per CTA and K block, else A and B
  static constexpr uint32_t kStage = MODE == kGatedBack ? 3 * kOperand + kOperand / 2 : kOperand + kOperandB;
  static constexpr int kStages = MODE == kGatedBack ? 3 : TN == 256 ? 6 : 8;
  static constexpr int kBuffers = MODE == kGatedBack ? 1 : 2;  // accumulators of 384 or TN columns in 512
  static constexpr uint32_t kSmem = kStage * kStages + kEpiWarps * kStaging + kBarBytes + 1024;
  static constexpr int kColumns = MODE == kGated || MODE == kGatedBack ? TN / 2 : TN;  // result columns per tile
  static constexpr int kChunks = kColumns / 32;             // epilogue chunks of 32 result columns
  static constexpr int kWarpChunks = (kChunks + 3) / 4;     // of a warp (four warps share a TMEM quadrant)
};

struct Problem {
  int a[2], b[2];                // tensor maps of the K segments
  int kb0, kb;                   // K blocks of the first segment, of both
  int m, n;                      // result
  int tiles_m, tiles_n;
  int first;                     // its first tile
  void *c;
  long long ldc;
};
struct Params {
  CUtensorMap map[kMaxMaps];
  Problem prob[kMaxProblems];
  int problems, items, maps;
  bool narrow;                   // tiles of 128 accumulator columns
  int whole, splits;             // tiles done by one work item each; parts of each tile after those
  void *c2;                      // du
  float *gu;                     // kept projections, see gu_index
  const float *a_scales, *b_scales, *bias;
  uint32_t *partial;             // raw sums: [tile - whole][part][kTileM][TN]
  WaitLimit wait;
};

struct Item {
  int prob, m0, n0, kb_begin, kb_end;
  uint32_t *partial;  // where raw sums go; nullptr: the item is a whole tile
};
template <int MODE, int TN>
__device__ __forceinline__ Item item_of(const Params &p, int it) {
  Item w;
  int tile = it, part = 0, parts = 1;
  w.partial = nullptr;
  if (it >= p.whole) {
    parts = p.splits;
    part = (it - p.whole) % parts;
    tile = p.whole + (it - p.whole) / parts;
    if (parts > 1) w.partial = p.partial + (size_t)(it - p.whole) * (kTileM * TN);
  }
  w.prob = 0;
#pragma unroll
  for (int i = 1; i < kMaxProblems; ++i)
    if (i < p.problems && tile >= p.prob[i].first) w.prob = i;
  const Problem &q = p.prob[w.prob];
  // groups of 8 row tiles, columns outer: the tiles in flight share their operands in L2
  tile -= q.first;
  const int group = tile / (8 * q.tiles_n), rows = min(8, q.tiles_m - 8 * group), t = tile - group * 8 * q.tiles_n;
  w.m0 = (8 * group + t % rows) * kTileM;
  w.n0 = (t / rows) * Shape<MODE, TN>::kColumns;
  w.kb_begin = 0;
  w.kb_end = q.kb;
  if (parts > 1) {  // kb < 2^24 and parts < 2^7: the products fit 31 bits
    w.kb_begin = q.kb * part / parts;
    w.kb_end = q.kb * (part + 1) / parts;
  }
  return w;
}

// Kept projections: g (which = 0) and u (1) of row r, hidden column c, blocks of 32
// rows so that a warp (lane = row) moves whole 128-byte lines straight from registers
__device__ __forceinline__ size_t gu_index(long long row, int c, int which, int hidden) {
  return ((size_t(row >> 5) * hidden + c) * 2 + which) * 32 + (row & 31);
}

// 64 bytes of each of the warp's 32 rows (lane = row) to C through the warp's staging,
// which turns them into stores of whole row segments. The 16-byte pieces of a staged
// row are permuted with the row: no bank conflicts either way. `cols`: columns left
// in the row from c on; `wide`: the rows of C start on 16-byte boundaries.
template <class O>
__device__ __forceinline__ void store_rows(unsigned char *stage, int lane, const Chunk<O, 16 / sizeof(O)> (&v)[4],
                                           O *c, long long ldc, int rows, int cols, bool wide) {
  constexpr int kPer = 16 / sizeof(O);
  auto slot = [&](int r, int piece) {
    return reinterpret_cast<O *>(stage + 64 * r + 16 * (piece ^ ((r >> 1) & 3)));
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) store_chunk<O, kPer>(slot(lane, i), v[i]);
  __syncwarp();
  if (wide && cols >= 4 * kPer) {  // 16 bytes a lane, 8 rows at a time
    const int piece = lane & 3;
    c += (lane >> 2) * ldc + piece * kPer;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 2);
      if (r < rows) store_chunk<O, kPer>(c + 8 * i * ldc, load_chunk<O, kPer>(slot(r, piece)));
    }
  } else {  // one element a lane: still whole row segments
    constexpr int kElems = 4 * kPer, kRows = 32 / kElems;
    const int e = lane % kElems, r0 = lane / kElems;
    c += r0 * ldc + e;
    if (e < cols)
#pragma unroll 8
      for (int r = r0; r < rows; r += kRows, c += kRows * ldc) *c = slot(r, e / kPer)[e % kPer];
  }
  __syncwarp();
}
// dg = dh u silu'(g), du = dh silu(g)
__device__ __forceinline__ void gradients(float g, float u, float dh, float &dg, float &du) {
  const float sg = sigmoid_f32(g);
  du = dh * (g * sg);
  dg = dh * u * (sg * fmaf(g, 1.0f - sg, 1.0f));
}

template <int MODE, class T, bool A_MN, bool B_MN, int TN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) k_dense(const __grid_constant__ Params p) {
  using S = Shape<MODE, TN>;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char *sm = smem_raw + (base - raw);
  unsigned char *staging = sm + S::kStage * S::kStages;
  unsigned char *bar_mem = staging + kEpiWarps * kStaging;
  const uint32_t bars = tc::smem_u32(bar_mem);
  auto full = [&](int s) { return bars + 8u * s; };                      // K block landed in both CTAs (leader)
  auto empty = [&](int s) { return bars + 8u * (kMaxStages + s); };      // MMAs done with it (both)
  auto acc_full = [&](int b) { return bars + 8u * (2 * kMaxStages + b); };       // accumulator complete (both)
  auto acc_empty = [&](int b) { return bars + 8u * (2 * kMaxStages + 2 + b); };  // read by both CTAs (leader)
  const uint32_t drain = bars + 8u * (2 * kMaxStages + 4);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bar_mem + 8 * (2 * kMaxStages + 5));
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(tc::cluster_rank());
  // for the end after a wait that gave up: K blocks that this CTA has fetched, and (leader) those that have been
  // multiplied and the items whose accumulator is complete
  volatile int *fetched = reinterpret_cast<volatile int *>(tmem_slot + 2);
  volatile int *multiplied = reinterpret_cast<volatile int *>(tmem_slot + 3);
  volatile int *finished = reinterpret_cast<volatile int *>(tmem_slot + 4);
  auto wait = [&](uint32_t bar, int parity, int where) {  // both CTAs learn of one that gives up
    const bool ok = tc::mbar_wait(bar, parity, abort_flag, p.wait.err, where, p.wait.cycles);
    if (!ok) tc::store_of_rank(abort_flag, rank ^ 1, 1);
    return ok;
  };
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  // the pair's n-th work item: its divisions and parameter reads are not on the path of every tile
  __shared__ Item table[kItemTable];
  for (int i = threadIdx.x; i < kItemTable && pair + i * pairs < p.items; i += kThreads)
    table[i] = item_of<MODE, TN>(p, pair + i * pairs);
  auto item = [&](int n) { return n < kItemTable ? table[n] : item_of<MODE, TN>(p, pair + n * pairs); };
  const int items = pair < p.items ? (p.items - 1 - pair) / pairs + 1 : 0;

  dependents_may_start();
  if (warp == 2 && lane < p.maps) tc::prefetch_map(&p.map[lane]);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      tc::mbar_init(full(s), 1);
      tc::mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(acc_full(b), 1);
      tc::mbar_init(acc_empty(b), 2 * kEpiWarps);
    }
    tc::mbar_init(drain, 1);
    *abort_flag = 0;
    *fetched = *multiplied = *finished = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc::smem_u32(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc::fence_before();
  __syncthreads();
  tc::cluster_sync();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_predecessors();

  if (warp == 0) {
    // ------------------------------------------------------------------- loads
    if (lane == 0) {
      int n = 0;
      bool ok = true;
      for (int it = 0; it < items && ok; ++it) {
        const Item w = item(it);
        const Problem &q = p.prob[w.prob];
        for (int kb = w.kb_begin; kb < w.kb_end; ++kb, ++n) {
          const int s = n % S::kStages;
          ok = wait(empty(s), ((n / S::kStages) & 1) ^ 1, 1);
          if (!ok) break;
          if (rank == 0) tc::mbar_expect_tx(full(s), 2 * S::kStage);
          const uint32_t bar = tc::at_leader(full(s)), dst = base + s * S::kStage;
          constexpr int kElems = MODE == kInt8 ? 128 : 64;  // of a K block
          if (MODE == kGated || MODE == kGatedBack) {
            const int k = kb * 64;
            tc::tma_load(dst, &p.map[0], k, w.m0 + 128 * rank, bar);                  // x
            tc::tma_load(dst + kOperand, &p.map[1 + rank], k, w.n0, bar);             // Wg | Wu
            if (MODE == kGatedBack) {
              tc::tma_load(dst + 2 * kOperand, &p.map[3], k, w.m0 + 128 * rank, bar); // dy
              tc::tma_load(dst + 3 * kOperand, &p.map[4], w.n0 + 64 * rank, k, bar);  // Wd
            }
          } else {
            const int seg = kb >= q.kb0 ? 1 : 0, k = (kb - (seg ? q.kb0 : 0)) * kElems;
            const CUtensorMap *a = &p.map[q.a[seg]], *b = &p.map[q.b[seg]];
            const int m = w.m0 + 128 * rank, c = w.n0 + TN / 2 * rank;
            if (A_MN) {
              tc::tma_load(dst, a, m, k, bar);
              tc::tma_load(dst + kOperand / 2, a, m + 64, k, bar);
            } else {
              tc::tma_load(dst, a, k, m, bar);
            }
            if (B_MN) {
              tc::tma_load(dst + kOperand, b, c, k, bar);
              if (TN == 256) tc::tma_load(dst + kOperand + kOperand / 2, b, c + 64, k, bar);
            } else {
              tc::tma_load(dst + kOperand, b, k, c, bar);
            }
          }
          *fetched = n + 1;
        }
      }
      // every release of a K block has reached this CTA before it may leave
      for (int i = max(0, n - S::kStages); i < n && ok; ++i)
        ok = wait(empty(i % S::kStages), (i / S::kStages) & 1, 6);
      // in the odd CTA also the leader's last signal. Not before: each wait is for one step of the pipeline, so that
      // its limit does not bound the whole kernel
      if (rank != 0 && ok) wait(drain, 0, 4);
    }
    __syncwarp();
  } else if (warp == 1) {
    // -------------------------------------------------------------------- MMAs
    if (rank == 0 && lane == 0) {
      constexpr bool kI8 = MODE == kInt8;
      constexpr uint32_t kAb = kI8 || std::is_same<T, __nv_bfloat16>::value ? 1 : 0;  // s8 / bf16, or f16
      constexpr uint32_t kId = tc::idesc(kI8 ? 2 : 1, kAb, A_MN, B_MN, TN);
      constexpr uint32_t kIdDh = tc::idesc(1, kAb, false, true, 128);
      int n = 0;
      bool ok = true;
      for (int done = 0; done < items && ok; ++done) {
        const Item w = item(done);
        const int buf = done % S::kBuffers;
        ok = wait(acc_empty(buf), ((done / S::kBuffers) & 1) ^ 1, 2);
        if (!ok) break;
        tc::fence_after();
        const uint32_t d = tmem + 256u * buf;
        for (int kb = w.kb_begin; kb < w.kb_end; ++kb, ++n) {
          const int s = n % S::kStages;
          ok = wait(full(s), (n / S::kStages) & 1, 3);
          if (!ok) break;
          tc::fence_after();
          const uint32_t a = base + s * S::kStage, b = a + kOperand;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint64_t da = A_MN ? tc::desc_mn(a + 2048 * ks, kOperand / 2) : tc::desc_k(a + 32 * ks);
            const uint64_t db = B_MN ? tc::desc_mn(b + 2048 * ks, kOperand / 2) : tc::desc_k(b + 32 * ks);
            tc::mma<kI8>(d, da, db, kId, kb > w.kb_begin || ks > 0);
            if (MODE == kGatedBack)
              tc::mma<false>(d + 256, tc::desc_k(a + 2 * kOperand + 32 * ks),
                             tc::desc_mn(a + 3 * kOperand + 2048 * ks, kOperand / 2), kIdDh,
                             kb > w.kb_begin || ks > 0);
          }
          tc::commit_pair(empty(s));
        }
        if (!ok) break;
        tc::commit_pair(acc_full(buf));
        *finished = done + 1;
      }
      // every MMA has completed
      *multiplied = n;
      tc::commit_pair(drain);
      wait(drain, 0, 4);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue
    // warp: TMEM lanes 32 (warp % 4) .. + 31, a quarter of the columns
    const int quad = warp & 3, part = (warp - 2) >> 2;
    unsigned char *stage = staging + (warp - 2) * kStaging;
    const uint32_t lanes = tmem + (uint32_t(32 * quad) << 16);
    for (int done = 0; done < items; ++done) {
      const Item w = item(done);
      const Problem &q = p.prob[w.prob];
      const int buf = done % S::kBuffers;
      if (!__all_sync(0xffffffffu, wait(acc_full(buf), (done / S::kBuffers) & 1, 5))) break;
      tc::fence_after();
      const uint32_t acc = lanes + 256u * buf;
      auto release = [&] {  // this warp has read its part of the accumulator
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_cluster(tc::at_leader(acc_empty(buf)));
      };
      const int row0 = w.m0 + 128 * rank + 32 * quad, rows = min(32, q.m - row0);
      constexpr int kPer = 16 / sizeof(T);
      const bool wide = (reinterpret_cast<uintptr_t>(q.c) | (q.ldc * sizeof(T))) % 16 == 0;
      if constexpr (MODE == kPlain || MODE == kInt8) {
        const bool split = w.partial != nullptr;
        const float sa = MODE == kInt8 && !split && lane < rows ? p.a_scales[row0 + lane] : 0.0f;
        for (int j = 0; j < S::kWarpChunks; ++j) {
          const int col = 32 * (S::kWarpChunks * part + j), c0 = w.n0 + col;
          uint32_t r[32];
          tc::tmem_ld32(acc + col, r);
          tc::wait_ld(r);
          if (j == S::kWarpChunks - 1) release();
          if (rows <= 0 || c0 >= q.n) continue;
          if (split) {  // raw 32-bit sums, float or int
            uint32_t *dst = w.partial + (128 * rank + 32 * quad) * TN + col;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              Chunk<float, 4> v[4];
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i / 4].e[i % 4] = __uint_as_float(r[16 * h + i]);
              store_rows<float>(stage, lane, v, reinterpret_cast<float *>(dst) + 16 * h, TN, rows, 16, true);
            }
            continue;
          }
          float sb = 0.0f, bias = 0.0f;
          if (MODE == kInt8 && c0 + lane < q.n) {
            sb = p.b_scales[c0 + lane];
            bias = p.bias ? p.bias[c0 + lane] : 0.0f;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // 32 columns of 2 bytes, or twice 16 of 4
            constexpr int kCols = 4 * kPer;
            if (h * kCols >= 32) break;
            Chunk<T, kPer> v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float f[kPer];
#pragma unroll
              for (int e = 0; e < kPer; ++e) {
                const int k = (h * kCols + i * kPer + e) % 32;
                f[e] = __uint_as_float(r[k]);
                if (MODE == kInt8)
                  f[e] = fmaf(float(int(r[k])) * sa, __shfl_sync(0xffffffffu, sb, k),
                              __shfl_sync(0xffffffffu, bias, k));
              }
              v[i] = to_chunk<T, kPer>(f);
            }
            store_rows<T>(stage, lane, v, static_cast<T *>(q.c) + row0 * q.ldc + c0 + h * kCols, q.ldc, rows,
                          q.n - c0 - h * kCols, wide);
          }
        }
      } else if constexpr (MODE == kKeptBack) {
        for (int j = 0; j < S::kWarpChunks; ++j) {
          const int col = 32 * (S::kWarpChunks * part + j), c0 = w.n0 + col;
          const bool live = rows > 0 && c0 < q.n;
          Chunk<T, kPer> out[4], out2[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float g[16], u[16];
            uint32_t dh[16];
            const float *gu = p.gu + gu_index(row0 + lane, c0 + 16 * h, 0, q.n);
            const int left = live ? q.n - c0 - 16 * h : 0;
            if (left >= 16) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                g[i] = __ldcs(gu + 64 * i);
                u[i] = __ldcs(gu + 64 * i + 32);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                g[i] = i < left ? gu[64 * i] : 0.0f;
                u[i] = i < left ? gu[64 * i + 32] : 0.0f;
              }
            }
            tc::tmem_ld16(acc + col + 16 * h, dh);
            tc::wait_ld(dh);
            if (j == S::kWarpChunks - 1 && h == 1) release();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float dg[8], du[8];
#pragma unroll
              for (int i = 0; i < 8; ++i)
                gradients(g[8 * k + i], u[8 * k + i], __uint_as_float(dh[8 * k + i]), dg[i], du[i]);
              out[2 * h + k] = to_chunk<T, 8>(dg);
              out2[2 * h + k] = to_chunk<T, 8>(du);
            }
          }
          if (!live) continue;
          const long long at = row0 * q.ldc + c0;
          store_rows<T>(stage, lane, out, static_cast<T *>(q.c) + at, q.ldc, rows, q.n - c0, wide);
          store_rows<T>(stage, lane, out2, static_cast<T *>(p.c2) + at, q.ldc, rows, q.n - c0, wide);
        }
      } else {
        const int col = 32 * part, c0 = w.n0 + col;
        const bool mine = part < S::kChunks, live = mine && rows > 0 && c0 < q.n;
        if (!mine) release();
        const long long at = row0 * q.ldc + c0;
        // only the 16-bit types have these modes
        using H = typename std::conditional<sizeof(T) == 2, T, __half>::type;
        Chunk<H, 8> out[4], out2[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!mine) break;
          uint32_t g[16], u[16], dh[16];
          tc::tmem_ld16(acc + col + 16 * h, g);
          tc::tmem_ld16(acc + TN / 2 + col + 16 * h, u);
          if (MODE == kGatedBack) tc::tmem_ld16(acc + 256 + col + 16 * h, dh);
          tc::wait_ld(g);
          tc::wait_ld(u);
          if (MODE == kGatedBack) tc::wait_ld(dh);
          if (h == 1) release();
          if (!live) continue;
          if (MODE == kGated && p.gu) {
            float *gu = p.gu + gu_index(row0 + lane, c0 + 16 * h, 0, q.n);
            const int left = q.n - c0 - 16 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (i < left) {
                __stcs(gu + 64 * i, __uint_as_float(g[i]));
                __stcs(gu + 64 * i + 32, __uint_as_float(u[i]));
              }
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float a[8], b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float gi = __uint_as_float(g[8 * k + i]), ui = __uint_as_float(u[8 * k + i]);
              if (MODE == kGated)
                a[i] = silu_f32(gi) * ui;
              else
                gradients(gi, ui, __uint_as_float(dh[8 * k + i]), a[i], b[i]);
            }
            out[2 * h + k] = to_chunk<H, 8>(a);
            if (MODE == kGatedBack) out2[2 * h + k] = to_chunk<H, 8>(b);
          }
        }
        if (!live) continue;
        store_rows<H>(stage, lane, out, static_cast<H *>(q.c) + at, q.ldc, rows, q.n - c0, wide);
        if (MODE == kGatedBack)
          store_rows<H>(stage, lane, out2, static_cast<H *>(p.c2) + at, q.ldc, rows, q.n - c0, wide);
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::cluster_sync();  // neither CTA leaves while the other may still signal it
  tc::fence_after();
  if (__builtin_expect(*abort_flag, 0)) {
    // A wait of either CTA gave up. All that the pair has started ends (with a limit) before TMEM is handed back
    // and shared memory is left: copies, MMAs and the signals of both. A K block's barrier counts the parts of both
    // CTAs, so the CTA that is behind answers for the parts that it has not fetched.
    int all = 0;  // K blocks that either has fetched
    if (threadIdx.x == 0) {
      const int mine = *fetched;
      all = max(mine, tc::load_of_rank(fetched, rank ^ 1));
#pragma unroll 1
      for (int n = mine; n < all; ++n) {
        const uint32_t bar = full(n % S::kStages);
        if (rank == 0)
          tc::mbar_expect_tx(bar, S::kStage);
        else
          tc::mbar_complete_tx(tc::at_leader(bar), S::kStage);
      }
    }
    __syncwarp();
    tc::cluster_sync();
    if (threadIdx.x == 0) {
      const long long t0 = clock64();
      const int through = tc::load_of_rank(multiplied, 0), tiles = tc::load_of_rank(finished, 0);
      auto settle = [&](uint32_t first, int begin, int end, int ring) {
#pragma unroll 1
        for (int i = max(0, begin); i < end; ++i) tc::mbar_settle(first + 8u * (i % ring), (i / ring) & 1, t0);
      };
      if (rank == 0) settle(full(0), through, all, S::kStages);
      settle(empty(0), through - S::kStages, through, S::kStages);
      settle(acc_full(0), tiles - S::kBuffers, tiles, S::kBuffers);
      settle(drain, 0, 1, 1);
    }
    __syncwarp();
    tc::cluster_sync();
    tc::fence_after();
  }
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// C of the split tiles = the sum of their parts, in order; 8-bit products get their
// scales here. A block does 4 or 8 rows of a tile, a thread 4 columns of one: latency
// counts, so there are many blocks and all parts of a thread are loaded together.
template <int MODE, class T, int TN>
__global__ void __launch_bounds__(256) k_join(const __grid_constant__ Params p) {
  dependents_may_start();
  constexpr int kQuads = TN / 4;  // of columns
  const Item w = item_of<MODE, TN>(p, p.whole + blockIdx.y * p.splits);
  const Problem &q = p.prob[w.prob];
  const int col = w.n0 + 4 * (threadIdx.x % kQuads);
  const int r = blockIdx.x * (256 / kQuads) + threadIdx.x / kQuads, row = w.m0 + r;
  if (col >= q.n || row >= q.m) return;
  wait_for_predecessors();
  float f[4] = {0, 0, 0, 0};
  int s[4] = {0, 0, 0, 0};
  const uint32_t *part = w.partial + (size_t)r * TN + col - w.n0;
  for (int k0 = 0; k0 < p.splits; k0 += 8) {
    uint4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k0 + k < p.splits) v[k] = *reinterpret_cast<const uint4 *>(part + (size_t)(k0 + k) * (kTileM * TN));
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k0 + k < p.splits) {
        const uint32_t e[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (MODE == kInt8)
            s[j] += int(e[j]);
          else
            f[j] += __uint_as_float(e[j]);
        }
      }
  }
  if (MODE == kInt8) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < q.n)
        f[j] = fmaf(float(s[j]) * p.a_scales[row], p.b_scales[col + j], p.bias ? p.bias[col + j] : 0.0f);
  }
  const Chunk<T, 4> out = to_chunk<T, 4>(f);
  T *dst = static_cast<T *>(q.c) + row * q.ldc + col;
  if ((reinterpret_cast<uintptr_t>(q.c) | (q.ldc * sizeof(T))) % (4 * sizeof(T)) == 0 && col + 4 <= q.n)
    store_chunk<T, 4>(dst, out);
  else
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < q.n) dst[j] = out.e[j];
}

// Operands copied to rows that start on 16-byte boundaries, all of a launch's in one
// kernel: a thread gathers 16 bytes of a padded row.
constexpr int kMaxRepack = 6;
struct Repack {
  struct Matrix {
    const void *src;
    void *dst;
    long long stride, first;  // first: its first 16-byte piece among all
    int cols, pieces;         // pieces of a row
  } m[kMaxRepack];
  int count;
  long long total;
};
template <class T>
__global__ void k_repack(const __grid_constant__ Repack a) {
  dependents_may_start();
  wait_for_predecessors();
  constexpr int kPer = 16 / sizeof(T);
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < a.total;
       i += (long long)gridDim.x * blockDim.x) {
    int k = 0;
#pragma unroll
    for (int j = 1; j < kMaxRepack; ++j)
      if (j < a.count && i >= a.m[j].first) k = j;
    const Repack::Matrix &m = a.m[k];
    const long long at = i - m.first;
    const long long r = a.total < (1LL << 31) ? uint32_t(at) / uint32_t(m.pieces) : at / m.pieces;
    const int c = int(at - r * m.pieces) * kPer;
    const T *src = static_cast<const T *>(m.src) + r * m.stride;
    Chunk<T, kPer> v{};
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (c + j < m.cols) v.e[j] = src[c + j];
    store_chunk<T, kPer>(static_cast<T *>(m.dst) + (r * m.pieces * kPer + c), v);
  }
}

// -------------------------------------------------------------------- host side
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult found;
    SO3_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !p) throw Error("cuTensorMapEncodeTiled: the driver does not have it");
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// Scratch handed out from the caller's workspace; with base == nullptr only counted.
class Scratch {
 public:
  explicit Scratch(void *base) : base_(static_cast<char *>(base)) {}
  void *take(long long bytes) {
    void *p = base_ + used_;
    used_ += (bytes + 255) / 256 * 256;
    return p;
  }
  long long used() const { return used_; }

 private:
  char *base_;
  long long used_ = 0;
};

// A row-major operand [rows][cols].
struct Operand {
  const void *data;
  long long stride;
  long long rows, cols;
};

// Builds and queues products; with `dry` only the scratch is counted, so that the
// workspace sizes come from the code that uses the workspace.
class Dense {
 public:
  Dense(void *workspace, int elem, cudaStream_t stream, bool dry)
      : scratch_(workspace), elem_(elem), stream_(stream), dry_(dry) {}
  Scratch &scratch() { return scratch_; }
  bool dry() const { return dry_; }

  // the operand as TMA reads it: in place, or copied to padded rows before the next run()
  Operand ready(Operand o) {
    const bool in_place = reinterpret_cast<uintptr_t>(o.data) % 16 == 0 &&
                          (o.rows == 1 || (o.stride * elem_ % 16 == 0 && o.stride >= o.cols));
    if (in_place) return o;
    const long long ld = padded(o.cols);
    void *p = scratch_.take(o.rows * ld * elem_);
    if (!dry_) {
      if (repack_.count == kMaxRepack) flush();
      const int pieces = int(ld * elem_ / 16);
      repack_.m[repack_.count++] = Repack::Matrix{o.data, p, o.stride, repack_.total, int(o.cols), pieces};
      repack_.total += o.rows * pieces;
    }
    return Operand{p, ld, o.rows, o.cols};
  }
  void flush() {
    if (repack_.count == 0) return;
    const unsigned grid = unsigned(std::min<long long>((repack_.total + 255) / 256, kSmCount * 32));
    if (elem_ == 1)
      launch(k_repack<uint8_t>, grid, 256, 0, stream_, repack_);
    else
      launch(k_repack<uint16_t>, grid, 256, 0, stream_, repack_);
    repack_.count = 0;
    repack_.total = 0;
  }
  long long padded(long long cols) const { return (cols * elem_ + 15) / 16 * 16 / elem_; }

  // A tensor map whose boxes are 128 bytes of `box_rows` rows.
  CUtensorMap map(const Operand &o, int box_rows) const {
    CUtensorMap m;
    const cuuint64_t dims[2] = {cuuint64_t(o.cols), cuuint64_t(o.rows)};
    const cuuint64_t stride[1] = {cuuint64_t((o.rows == 1 ? padded(o.cols) : o.stride) * elem_)};
    const cuuint32_t box[2] = {cuuint32_t(128 / elem_), cuuint32_t(box_rows)}, step[2] = {1, 1};
    const CUresult r = encode_tiled()(
        &m, elem_ == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2,
        const_cast<void *>(o.data), dims, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw Error("cuTensorMapEncodeTiled failed with " + std::to_string(int(r)));
    return m;
  }

  // Work items of the problems. Tiles are narrow where 256 columns would give half of
  // the pairs or fewer a tile, unless the contraction is long enough to keep all pairs
  // busy in parts (they then read a third less). The tiles after the last whole wave
  // are split along K where that saves more than the join costs: a K block takes a pair
  // 0.3 us, a join with its launch 5 (narrow tiles) to 7 us.
  template <int MODE>
  void plan(Params &p, bool may_split) {
    long long tiles = count<MODE, 256>(p);
    int kb = 1 << 30;
    for (int i = 0; i < p.problems; ++i) kb = std::min(kb, p.prob[i].kb);
    p.narrow = MODE != kGatedBack && 2 * tiles <= kPairs && (!may_split || tiles * kb < 24 * kPairs);
    if (p.narrow) tiles = count<MODE, 128>(p);
    if (tiles > (1LL << 30)) throw Error("feed-forward layers: the product has too many tiles");
    const int rest = int(tiles % kPairs);
    int splits = may_split && rest > 0 ? std::max(1, std::min(kPairs / rest, kb / 8)) : 1;
    if (kb - kb / splits < (p.narrow ? 16 : 24)) splits = 1;
    p.splits = splits;
    p.whole = int(tiles) - (p.splits > 1 ? rest : 0);
    p.items = p.whole + (p.splits > 1 ? rest * p.splits : 0);
    p.partial = p.splits > 1 ? static_cast<uint32_t *>(scratch_.take((long long)rest * p.splits * kTileM *
                                                                    (p.narrow ? 128 : 256) * 4))
                             : nullptr;
  }
  template <int MODE, int TN>
  static long long count(Params &p) {
    long long tiles = 0;
    for (int i = 0; i < p.problems; ++i) {
      Problem &q = p.prob[i];
      q.tiles_m = (q.m - 1) / kTileM + 1;
      q.tiles_n = (q.n - 1) / Shape<MODE, TN>::kColumns + 1;
      q.first = int(std::min<long long>(tiles, 1 << 30));
      tiles += (long long)q.tiles_m * q.tiles_n;
    }
    return tiles;
  }

  template <int MODE, class T, bool A_MN, bool B_MN>
  void run(Params &p) {
    flush();
    if constexpr (MODE != kGatedBack) {
      if (p.narrow) return run_tiles<MODE, T, A_MN, B_MN, 128>(p);
    }
    run_tiles<MODE, T, A_MN, B_MN, 256>(p);
  }
  template <int MODE, class T, bool A_MN, bool B_MN, int TN>
  void run_tiles(Params &p) {
    using S = Shape<MODE, TN>;
    allow_dynamic_smem(reinterpret_cast<const void *>(&k_dense<MODE, T, A_MN, B_MN, TN>), S::kSmem);
    p.wait = wait_limit();
    launch(k_dense<MODE, T, A_MN, B_MN, TN>, 2 * std::min(kPairs, p.items), kThreads, S::kSmem, stream_, p);
    if constexpr (MODE == kPlain || MODE == kInt8) {
      if (p.splits == 1) return;
      const int rows = 256 / (TN / 4);  // of a block
      launch(k_join<MODE, T, TN>, dim3(kTileM / rows, (p.items - p.whole) / p.splits), 256, 0, stream_, p);
    }
  }

 private:
  Scratch scratch_;
  int elem_;
  cudaStream_t stream_;
  bool dry_;
  Repack repack_{};
};

int blocks_of(long long k, int per) { return int((k + per - 1) / per); }

template <class F>
void by_half(int dtype, F &&f) {
  if (dtype == SO3LR_BFLOAT16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}

// ------------------------------------------------------------------ 8-bit product
template <class O>
void int8_linear(Dense &d, const so3lr_int8_linear_args &a) {
  Params p{};
  const Operand x = d.ready(Operand{a.a, a.a_stride, a.rows, a.k}), w = d.ready(Operand{a.b, a.b_stride, a.n, a.k});
  p.problems = 1;
  p.a_scales = a.a_scales;
  p.b_scales = a.b_scales;
  p.bias = a.bias;
  Problem &q = p.prob[0];
  q.a[0] = 0;
  q.b[0] = 1;
  q.kb = q.kb0 = blocks_of(a.k, 128);
  q.m = int(a.rows);
  q.n = int(a.n);
  q.c = a.y;
  q.ldc = a.y_stride;
  d.plan<kInt8>(p, true);
  if (d.dry()) return;
  p.maps = 2;
  p.map[0] = d.map(x, 128);
  p.map[1] = d.map(w, p.narrow ? 64 : 128);
  d.run<kInt8, O, false, false>(p);
}

// ------------------------------------------------------------------- feed-forward
// Keeping g and u costs 16 bytes of HBM traffic an element, computing them again 4
// width operations: at this card's 1.6 PFLOP/s and 6.5 TB/s the two are even near a
// width of 1024.
bool keeps(long long width) { return width >= 1024; }

template <class T>
void feed_forward(Dense &d, const so3lr_feed_forward_args &a) {
  const Operand x = d.ready(Operand{a.x, a.x_stride, a.rows, a.width});
  const Operand g = d.ready(Operand{a.w_gate, a.w_gate_stride, a.hidden, a.width});
  const Operand u = d.ready(Operand{a.w_up, a.w_up_stride, a.hidden, a.width});
  const Operand w = d.ready(Operand{a.w_down, a.w_down_stride, a.width, a.hidden});
  Operand h{a.h, a.hidden, a.rows, a.hidden};
  if (!a.h) {
    h.stride = d.padded(a.hidden);
    h.data = d.scratch().take(a.rows * h.stride * 2);
  }
  {
    Params p{};
    p.problems = 1;
    Problem &q = p.prob[0];
    q.kb = q.kb0 = blocks_of(a.width, 64);
    q.m = int(a.rows);
    q.n = int(a.hidden);
    q.c = const_cast<void *>(h.data);
    q.ldc = h.stride;
    p.gu = a.gu;
    d.plan<kGated>(p, false);
    if (!d.dry()) {
      p.maps = 3;
      p.map[0] = d.map(x, 128);
      p.map[1] = d.map(g, p.narrow ? 64 : 128);
      p.map[2] = d.map(u, p.narrow ? 64 : 128);
      d.run<kGated, T, false, false>(p);
    }
  }
  const Operand hr = d.ready(h);
  Params p{};
  p.problems = 1;
  Problem &q = p.prob[0];
  q.a[0] = 0;
  q.b[0] = 1;
  q.kb = q.kb0 = blocks_of(a.hidden, 64);
  q.m = int(a.rows);
  q.n = int(a.width);
  q.c = a.y;
  q.ldc = a.y_stride;
  d.plan<kPlain>(p, true);
  if (d.dry()) return;
  p.maps = 2;
  p.map[0] = d.map(hr, 128);
  p.map[1] = d.map(w, p.narrow ? 64 : 128);
  d.run<kPlain, T, false, false>(p);
}

template <class T>
void feed_forward_backward(Dense &d, const so3lr_feed_forward_backward_args &a) {
  const Operand x = d.ready(Operand{a.x, a.x_stride, a.rows, a.width});
  const Operand dy = d.ready(Operand{a.dy, a.dy_stride, a.rows, a.width});
  const Operand g = d.ready(Operand{a.w_gate, a.w_gate_stride, a.hidden, a.width});
  const Operand u = d.ready(Operand{a.w_up, a.w_up_stride, a.hidden, a.width});
  const Operand w = d.ready(Operand{a.w_down, a.w_down_stride, a.width, a.hidden});
  const Operand h = d.ready(Operand{a.h, a.hidden, a.rows, a.hidden});
  const long long ld = d.padded(a.hidden);
  Operand dg{d.scratch().take(a.rows * ld * 2), ld, a.rows, a.hidden}, du = dg;
  du.data = d.scratch().take(a.rows * ld * 2);
  {
    Params p{};
    p.problems = 1;
    Problem &q = p.prob[0];
    q.kb = q.kb0 = blocks_of(a.width, 64);
    q.m = int(a.rows);
    q.n = int(a.hidden);
    q.c = const_cast<void *>(dg.data);
    q.ldc = ld;
    p.c2 = const_cast<void *>(du.data);
    if (a.gu) {
      p.gu = const_cast<float *>(a.gu);
      q.a[0] = 0;
      q.b[0] = 1;
      d.plan<kKeptBack>(p, false);
    } else {
      d.plan<kGatedBack>(p, false);
    }
    if (a.gu && !d.dry()) {
      p.maps = 2;
      p.map[0] = d.map(dy, 128);
      p.map[1] = d.map(w, 64);
      d.run<kKeptBack, T, false, true>(p);
    } else if (!d.dry()) {
      p.maps = 5;
      p.map[0] = d.map(x, 128);
      p.map[1] = d.map(g, 128);
      p.map[2] = d.map(u, 128);
      p.map[3] = d.map(dy, 128);
      p.map[4] = d.map(w, 64);
      d.run<kGatedBack, T, false, false>(p);
    }
  }
  {  // dx = dg Wg + du Wu: one contraction over both
    Params p{};
    p.problems = 1;
    Problem &q = p.prob[0];
    q.a[0] = 0;
    q.a[1] = 1;
    q.b[0] = 2;
    q.b[1] = 3;
    q.kb0 = blocks_of(a.hidden, 64);
    q.kb = 2 * q.kb0;
    q.m = int(a.rows);
    q.n = int(a.width);
    q.c = a.dx;
    q.ldc = a.dx_stride;
    d.plan<kPlain>(p, true);
    if (!d.dry()) {
      p.maps = 4;
      p.map[0] = d.map(dg, 128);
      p.map[1] = d.map(du, 128);
      p.map[2] = d.map(g, 64);
      p.map[3] = d.map(u, 64);
      d.run<kPlain, T, false, true>(p);
    }
  }
  // the three weight gradients, contracted over the rows, in one launch
  Params p{};
  p.problems = 3;
  for (int i = 0; i < 3; ++i) {
    Problem &q = p.prob[i];
    q.a[0] = i;              // dg, du, dy
    q.b[0] = i < 2 ? 3 : 4;  // x, x, h
    q.kb = q.kb0 = blocks_of(a.rows, 64);
    q.m = int(i < 2 ? a.hidden : a.width);
    q.n = int(i < 2 ? a.width : a.hidden);
    q.c = i == 0 ? a.dw_gate : i == 1 ? a.dw_up : a.dw_down;
    q.ldc = q.n;
  }
  d.plan<kPlain>(p, true);
  if (d.dry()) return;
  p.maps = 5;
  p.map[0] = d.map(dg, 64);
  p.map[1] = d.map(du, 64);
  p.map[2] = d.map(dy, 64);
  p.map[3] = d.map(x, 64);
  p.map[4] = d.map(h, 64);
  d.run<kPlain, T, true, true>(p);
}

template <class A, class F>
long long dry_run(const A &a, int elem, F &&f) {
  if (a.rows == 0) return 0;
  Dense d(nullptr, elem, nullptr, true);
  f(d);
  return d.scratch().used();
}

}  // namespace

// Where a kernel whose wait gave up says so: a word for each device in page-locked host
// memory that all of them can write.
int *gave_up_flag() {
  constexpr int kMaxDevices = 64;
  static int *flags = [] {
    // allowed while another stream of the thread is being captured: it is no stream operation
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    SO3_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    void *p = nullptr;
    const cudaError_t e = cudaHostAlloc(&p, kMaxDevices * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
    cudaThreadExchangeStreamCaptureMode(&mode);
    SO3_CUDA(e);
    std::memset(p, 0, kMaxDevices * sizeof(int));
    return static_cast<int *>(p);
  }();
  int device = 0;
  SO3_CUDA(cudaGetDevice(&device));
  if (device >= kMaxDevices) throw Error("feed-forward layers: more than 64 devices");
  return flags + device;
}
void check_gave_up() {
  const int where = *static_cast<volatile int *>(gave_up_flag());
  if (where) throw Error(gave_up_message(where) + "; so3lr_layers_status clears this");
}
int take_gave_up() { return __atomic_exchange_n(gave_up_flag(), 0, __ATOMIC_SEQ_CST); }
static std::atomic<long long> g_wait_cycles{tc::kWaitCycles};
WaitLimit wait_limit() { return WaitLimit{gave_up_flag(), g_wait_cycles.load(std::memory_order_relaxed)}; }
void set_wait_limit(long long cycles) { g_wait_cycles = cycles > 0 ? cycles : tc::kWaitCycles; }
std::string gave_up_message(int where) {
  return "feed-forward layers: a kernel of an earlier call on this device gave up waiting (stage " +
         std::to_string(where) + "); the results of that call and of those after it are not valid";
}

long long int8_linear_bytes(const so3lr_int8_linear_args &a) {
  if (few_rows(a)) return 0;
  return dry_run(a, 1, [&](Dense &d) { int8_linear<float>(d, a); });
}
void launch_int8_linear(const so3lr_int8_linear_args &a, void *workspace, cudaStream_t s) {
  if (few_rows(a)) return launch_int8_linear_few(a, s);
  Dense d(workspace, 1, s, false);
  if (a.out_dtype == SO3LR_FLOAT32)
    int8_linear<float>(d, a);
  else
    by_half(a.out_dtype, [&](auto t) { int8_linear<decltype(t)>(d, a); });
}

long long feed_forward_keep(const so3lr_feed_forward_args &a) {
  so3lr_feed_forward_args plain = a;
  plain.gu = nullptr;
  return !few_rows(plain) && keeps(a.width) ? (a.rows + 31) / 32 * 32 * a.hidden * 8 : 0;
}
// The hidden layer of a few rows: its two parts with the same strides, on 16-byte
// boundaries (or contiguous, where the first is the caller's).
static long long few_stride(const so3lr_feed_forward_args &a) { return a.h ? a.hidden : (a.hidden + 7) / 8 * 8; }
static long long few_part(const so3lr_feed_forward_args &a) {
  return (a.rows * few_stride(a) * 2 + 255) / 256 * 256;
}
long long feed_forward_bytes(const so3lr_feed_forward_args &a) {
  if (few_rows(a)) return few_part(a) * (a.h ? 1 : 2);
  return dry_run(a, 2, [&](Dense &d) { feed_forward<__half>(d, a); });
}
void launch_feed_forward(const so3lr_feed_forward_args &a, void *workspace, cudaStream_t s) {
  if (few_rows(a)) {
    char *scratch = static_cast<char *>(workspace);
    return launch_feed_forward_few(a, a.h ? a.h : scratch + few_part(a), few_stride(a), scratch, s);
  }
  Dense d(workspace, 2, s, false);
  by_half(a.dtype, [&](auto t) { feed_forward<decltype(t)>(d, a); });
}

long long feed_forward_backward_bytes(const so3lr_feed_forward_backward_args &a) {
  return dry_run(a, 2, [&](Dense &d) { feed_forward_backward<__half>(d, a); });
}
void launch_feed_forward_backward(const so3lr_feed_forward_backward_args &a, void *workspace, cudaStream_t s) {
  if (a.rows == 0) {
    const std::size_t bytes = std::size_t(a.hidden) * a.width * 2;
    for (void *w : {a.dw_gate, a.dw_up, a.dw_down}) SO3_CUDA(cudaMemsetAsync(w, 0, bytes, s));
    return;
  }
  Dense d(workspace, 2, s, false);
  by_half(a.dtype, [&](auto t) { feed_forward_backward<decltype(t)>(d, a); });
}

}  // namespace so3lr_b200
