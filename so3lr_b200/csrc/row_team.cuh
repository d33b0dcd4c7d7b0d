// Rows of the row kernels (rows.cu, sandwich.cu): the threads that hold one, where its
// elements lie in them, rows through a ring in shared memory, and how a call chooses
// among these.
#pragma once

#include <algorithm>

#include "layers_common.cuh"
#include "model_host.hpp"
#include "tensor_core.cuh"

namespace so3lr_b200 {
namespace {

constexpr int kTeamThreads = 256;  // of a block whose rows belong to parts of a warp

// The threads of one row: LANES of a warp, or the whole block (LANES = 0). Reductions
// run in a fixed order and return the same value to every thread of the row.
template <int LANES>
struct RowTeam {
  int t, size;
  __device__ RowTeam() : t(LANES ? threadIdx.x % LANES : threadIdx.x), size(LANES ? LANES : blockDim.x) {}
  static __device__ __forceinline__ float add(float v) {
#pragma unroll
    for (int o = (LANES ? LANES : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  static __device__ __forceinline__ uint32_t largest(uint32_t v) {
    if (!LANES || LANES == 32) return __reduce_max_sync(0xffffffffu, v);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = ::max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
  // slot: 32 elements of shared memory that no other pending reduction uses
  // the sum of v; bits becomes the row's largest
  __device__ __forceinline__ float sum_and_max(float v, uint32_t &bits, float *slot, uint32_t *slot_max) const {
    v = add(v);
    bits = largest(bits);
    if (LANES) return v;
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) {
      slot[threadIdx.x >> 5] = v;
      slot_max[threadIdx.x >> 5] = bits;
    }
    __syncthreads();
    float total = 0.0f;
    for (int i = 0; i < warps; ++i) {
      total += slot[i];
      bits = ::max(bits, slot_max[i]);
    }
    return total;
  }
  __device__ __forceinline__ float sum(float v, float *slot) const {
    v = add(v);
    if (LANES) return v;
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    float total = 0.0f;
    for (int i = 0; i < warps; ++i) total += slot[i];
    return total;
  }
  __device__ __forceinline__ float2 sum2(float a, float b, float2 *slot) const {
    a = add(a);
    b = add(b);
    if (LANES) return make_float2(a, b);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 total = make_float2(0.0f, 0.0f);
    for (int i = 0; i < warps; ++i) {
      total.x += slot[i].x;
      total.y += slot[i].y;
    }
    return total;
  }
  __device__ __forceinline__ float3 sum3(float a, float b, float c, float *slot, float2 *slot2) const {
    a = add(a);
    b = add(b);
    c = add(c);
    if (LANES) return make_float3(a, b, c);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) {
      slot[threadIdx.x >> 5] = a;
      slot2[threadIdx.x >> 5] = make_float2(b, c);
    }
    __syncthreads();
    float3 total = make_float3(0.0f, 0.0f, 0.0f);
    for (int i = 0; i < warps; ++i) {
      total.x += slot[i];
      total.y += slot2[i].x;
      total.z += slot2[i].y;
    }
    return total;
  }
  __device__ __forceinline__ uint32_t max(uint32_t v, uint32_t *slot) const {
    v = largest(v);
    if (LANES) return v;
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    uint32_t top = 0;
    for (int i = 0; i < warps; ++i) top = ::max(top, slot[i]);
    return top;
  }
};
// The row of this thread's team; `live`: it exists. A team past the last row goes
// through the last one again without storing, so that whole warps stay together.
template <int LANES>
__device__ __forceinline__ long long team_row(long long rows, bool &live) {
  constexpr int kLanes = LANES ? LANES : 1;
  const long long row =
      LANES ? (long long)blockIdx.x * (kTeamThreads / kLanes) + threadIdx.x / kLanes : (long long)blockIdx.x;
  live = row < rows;
  return live ? row : rows - 1;
}

// Which elements of a row a thread holds: chunks of VEC, from the row's start or (SHIFT)
// from the first boundary of VEC elements in it; then what is left before the first and
// after the last whole chunk, fewer than VEC elements each, goes one to a thread. So no
// chunk is looked at element by element, and rows of any start and length cost little
// more than those on the boundaries.
template <bool SHIFT, int VEC>
struct Span {
  int first, width, edge;  // of the first chunk; edge: this thread's single element, -1 for none
  template <class T>
  __device__ Span(const T *row, int w, int t) : first(0), width(w), edge(-1) {
    if (!SHIFT) return;
    first = min(int((VEC - reinterpret_cast<uintptr_t>(row) / sizeof(T) % VEC) % VEC), w);
    const int e = t < first ? t : t + (w - first) / VEC * VEC;
    if (e < w && t < 2 * VEC) edge = e;
  }
  __device__ __forceinline__ int at(int chunk) const { return first + chunk * VEC; }
  __device__ __forceinline__ bool holds(int c) const { return SHIFT ? c + VEC <= width : c < width; }
};
// a chunk of what may lie on other boundaries than the row that the span is of
template <bool SHIFT, class T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> load_apart(const T *p) {
  if (!SHIFT) return load_chunk<T, VEC>(p);
  Chunk<T, VEC> v;
#pragma unroll
  for (int i = 0; i < VEC; ++i) v.e[i] = p[i];
  return v;
}
template <bool SHIFT, class T, int VEC>
__device__ __forceinline__ void store_apart(T *p, const Chunk<T, VEC> &v) {
  if (!SHIFT) {
    store_chunk<T, VEC>(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) p[i] = v.e[i];
}

// A ring of rows in shared memory, filled by bulk copies: what is in flight costs no
// registers, so a block that walks over rows keeps the memory system busy while it
// reduces and writes the current one. One block barrier after the last read of a
// stage, thread 0 may refill it. A wait that gives up marks its row; the block leaves
// its loop after that row's barrier, where every thread sees the mark, and not before
// the copies in flight have landed.
struct RowRing {
  uint32_t bars, buffer, stage_bytes;
  int stages;
  unsigned char *mem;
  WaitLimit limit;
  volatile int *abort_flag;  // 1 + the row of this block at which a wait gave up

  __device__ RowRing(unsigned char *smem, uint32_t bytes, int nstages, const WaitLimit &l)
      : stage_bytes(bytes), stages(nstages), mem(smem + 128), limit(l) {
    bars = tc::smem_u32(smem);
    buffer = bars + 128;
    abort_flag = reinterpret_cast<volatile int *>(smem + 120);
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) tc::mbar_init(bars + 8 * i, 1);
      *abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
  }
  __device__ const unsigned char *stage(int i) const { return mem + (i % stages) * stage_bytes; }
  // waits for the i-th row of this block
  __device__ void wait(int i) const {
    tc::mbar_wait(bar(i), (i / stages) & 1, abort_flag, limit.err, 7, limit.cycles, i + 1);
  }
  // after the barrier of the i-th row: whether a thread gave up waiting for it (a later row's mark does not count,
  // so all threads agree)
  __device__ bool gave_up(int i) const {
    const int at = *abort_flag;
    return at != 0 && at <= i + 1;
  }
  // thread 0, at the loop's end: the copies of rows i and on, of `rows`, have landed
  __device__ void settle(int i, int rows) const {
    const long long t0 = clock64();
    for (const int end = min(i + stages, rows); i < end; ++i) tc::mbar_settle(bar(i), (i / stages) & 1, t0);
  }
  // thread 0: the copies of the i-th row
  __device__ uint32_t expect(int i, uint32_t bytes) const {
    tc::mbar_expect_tx(bars + 8 * (i % stages), bytes);
    return buffer + (i % stages) * stage_bytes;
  }
  __device__ uint32_t bar(int i) const { return bars + 8 * (i % stages); }
};
constexpr int kRingHeader = 128, kRingStages = 8;

// ------------------------------------------------------------------ dispatch
bool aligned(const void *p, long long stride, int size, int bytes) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && (stride * size) % bytes == 0);
}

// Threads that hold a row of `width` elements, `per` of them each.
int row_threads(long long width, int per) { return int((width + 32LL * per - 1) / (32LL * per)) * 32; }

// How a thread's elements lie: 16-byte chunks from the row's start (kWide) or from the
// first boundary in it (kShifted, see Span), or single elements.
enum Path { kScalar, kWide, kShifted };
constexpr int chunk_of(Path path, int size) { return path == kScalar ? 1 : 16 / size; }
struct RowTensors {  // of one row: all that is moved in chunks of the element type
  int size;
  bool any = false, same = true;
  uintptr_t base = 0, step = 0;
  void add(const void *p, long long stride) {
    if (!p) return;
    const uintptr_t b = reinterpret_cast<uintptr_t>(p) % 16, t = uintptr_t(stride * size) % 16;
    if (any && (b != base || t != step)) same = false;
    any = true;
    base = b;
    step = t;
  }
  // `rest_aligned`: what is moved beside them in chunks lies on its boundaries
  Path path(long long width, bool rest_aligned) const {
    if (!same) return kScalar;
    return base == 0 && step == 0 && width * size % 16 == 0 && rest_aligned ? kWide : kShifted;
  }
};

// How a row is held: lanes of a warp (0: a block) and elements a thread. In a warp as
// few lanes as hold it with 8 elements each, then 16; a block of 64 threads would be
// bound by the rate at which blocks start (512 bfloat16 to 8 bits: 69 us, 31 in a warp).
// Longer rows: their products 8 a thread where they are on the boundaries, 16 beyond 4096
// and off the boundaries (1024: 41 us, 66 with 32 in a warp; 3001: 56 with 16, 63 with 8),
// the gradient off them 8 (71 and 191). Rows that become 8 bits issue more than they
// move and take fuller threads: 32 in a warp up to 1024 on the boundaries, above 32
// in a block for the gate (2048: 27 us, 33 with 16), 16 for the norm (31, 42 with 32) and
// for both off them (1003: 44 and 43 us, 49 and 52 in a warp). Bfloat16 rows, 33.5 M elements.
enum RowOp { kNorm, kNormBack, kNorm8, kGate8 };
struct Hold {
  int lanes, per;
};
constexpr Hold hold(long long width, Path path, int size, RowOp op) {
  if (path != kScalar) {
    // rows off the boundaries: their edges take up to 2 (16 / size - 1) threads
    if (width <= 64 && (path == kWide || size == 4)) return {8, 8};
    if (width <= 128) return {16, 8};
  }
  if (width <= 512) return {32, width <= 256 ? 8 : 16};
  if (path == kScalar) return {0, width <= 8192 ? 8 : op == kGate8 && width > 16384 ? 32 : 16};
  if (op == kNorm8 || op == kGate8) {
    if (path == kShifted) return {0, 16};
    return width <= 1024 ? Hold{32, 32} : Hold{0, op == kGate8 ? 32 : 16};
  }
  return {0, width <= (path == kShifted && op == kNorm ? 1024 : 4096) ? 8 : 16};
}
// Whether a call reaches the kernels that hold a row so. The widths are those at which
// hold() changes, each the widest of its kind.
constexpr bool reached(Path path, int size, RowOp op, int lanes, int per) {
  for (const int width : {64, 128, 256, 512, 1024, 4096, 8192, 16384, 32768}) {
    if (width > (op == kGate8 ? 32768 : 16384)) continue;
    if (op == kGate8 && path != kWide && (path == kScalar) != (width > 16384)) continue;  // launch_gate_int8
    if (op == kNormBack && path == kWide && width > 512 && width <= 8192) continue;       // backward_ring
    const Hold h = hold(width, path, size, op);
    if (h.lanes == lanes && h.per == per) return true;
  }
  return false;
}
// f(std::integral_constant lanes, std::integral_constant per) for h; kernels are compiled
// for those that a call reaches
template <Path PATH, int SIZE, RowOp OP, class F>
void by_hold(const Hold &h, F &&f) {
  bool found = false;
  auto lanes_per = [&](auto lanes, auto per) {
    if constexpr (reached(PATH, SIZE, OP, decltype(lanes)::value, decltype(per)::value))
      if (h.lanes == lanes && h.per == per) {
        found = true;
        f(lanes, per);
      }
  };
  using std::integral_constant;
  lanes_per(integral_constant<int, 8>{}, integral_constant<int, 8>{});
  lanes_per(integral_constant<int, 16>{}, integral_constant<int, 8>{});
  lanes_per(integral_constant<int, 32>{}, integral_constant<int, 8>{});
  lanes_per(integral_constant<int, 32>{}, integral_constant<int, 16>{});
  lanes_per(integral_constant<int, 32>{}, integral_constant<int, 32>{});
  lanes_per(integral_constant<int, 0>{}, integral_constant<int, 8>{});
  lanes_per(integral_constant<int, 0>{}, integral_constant<int, 16>{});
  lanes_per(integral_constant<int, 0>{}, integral_constant<int, 32>{});
  if (!found) throw Error("feed-forward layers: no kernel holds such a row");
}
template <class F>
void by_path(Path path, F &&f) {
  if (path == kWide)
    f(std::integral_constant<Path, kWide>{});
  else if (path == kShifted)
    f(std::integral_constant<Path, kShifted>{});
  else
    f(std::integral_constant<Path, kScalar>{});
}
// block and grid of one row a team
dim3 team_block(const Hold &h, long long width) {
  return h.lanes ? kTeamThreads : unsigned(row_threads(width, h.per));
}
dim3 team_grid(const Hold &h, long long rows) {
  const long long teams = h.lanes ? kTeamThreads / h.lanes : 1;
  return unsigned((rows + teams - 1) / teams);
}

template <class F>
void by_type(int dtype, F &&f) {
  if (dtype == SO3LR_FLOAT32)
    f(float{});
  else if (dtype == SO3LR_BFLOAT16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}
template <class T, class F>
void by_weight(int dtype, int weight_dtype, F &&f) {
  if (weight_dtype == SO3LR_FLOAT32 && dtype != SO3LR_FLOAT32)
    f(float{});
  else
    f(T{});
}

// Blocks of a kernel that walks over rows
int walking_blocks(const Hold &h, long long rows, long long width) {
  const int per_sm = h.lanes ? 4 : std::max(1, std::min(8, 1024 / row_threads(width, h.per)));
  return int(std::min<long long>(team_grid(h, rows).x, (long long)kSmCount * per_sm));
}

// Ring of a kernel that walks over rows: as many blocks an SM as its registers hold
// (`resident` threads), shared memory for up to kRingStages rows each. stages < 2: the
// row is too long.
struct RingPlan {
  int grid, stages, smem;
};
RingPlan ring_plan(long long rows, int threads, int resident, int depth, long long row_bytes) {
  // not more blocks than have room for `depth` rows each
  const int per_sm = int(std::max<long long>(
      1, std::min<long long>(std::min(16, resident / threads), 220 * 1024 / (depth * row_bytes + 2048 + kRingHeader))));
  const long long room = 220 * 1024 / per_sm - 2048 - kRingHeader;  // 2 KB: static and reserved shared memory
  RingPlan p;
  p.grid = int(std::min<long long>(rows, (long long)kSmCount * per_sm));
  p.stages = int(std::min<long long>(kRingStages, room / row_bytes));
  p.smem = int(kRingHeader + p.stages * row_bytes);
  return p;
}

}  // namespace
}  // namespace so3lr_b200
