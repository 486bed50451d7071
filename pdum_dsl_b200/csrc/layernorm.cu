// Layer norm for training: the forward with the rows' statistics, and the
// gradients of the input, the scale and the shift.  f32 or bf16 rows; every
// sum and statistic in f32.
//
//   mean = sum(x) / C      rstd = 1 / sqrt(sum((x - mean)^2) / C + eps)
//   z = (x - mean) rstd    y = z g + b
//   dx = rstd (dz - sum(dz) / C - z sum(dz z) / C)   with dz = dy g
//   dg = sum over rows of dy z      db = sum over rows of dy
//
// Both directions are HBM-bound: the forward reads x and writes y, the backward
// reads x and dy and writes dx, each once.  A row belongs to TPR threads, which
// keep it in registers between its two reductions.  On a B200, calls in a row, against a
// copy of the same bytes: forward 8192 x 4096 bf16 26.6 us (24.7), gradients with the
// weights' 8192 x 4096 f32 70 us (67), 262144 x 128 bf16 38 us (37); rows too long for
// one block lie on a cluster, from a cold L2: gradients 2048 x 16384 bf16 50 us, forward
// 1000 x 32768 39.
#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace pdb {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// VEC consecutive elements, moved as one access of sizeof(T) * VEC bytes.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

__device__ __forceinline__ float param_at(const void* p, int bf16, int64_t c) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]) : static_cast<const float*>(p)[c];
}
// VEC consecutive parameters from c on; vec: the vectors are 16-byte aligned and so is element c.
template <int VEC>
__device__ __forceinline__ void params_at(const void* p, int bf16, int vec, int64_t c, float (&out)[VEC]) {
  if (VEC > 1 && vec && !bf16) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + c + i));
      out[i] = q.x, out[i + 1] = q.y, out[i + 2] = q.z, out[i + 3] = q.w;
    }
  } else if (VEC == 8 && vec) {
    const Pack<__nv_bfloat16, VEC> q =
        *reinterpret_cast<const Pack<__nv_bfloat16, VEC>*>(static_cast<const __nv_bfloat16*>(p) + c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = to_f32(q.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = param_at(p, bf16, c + i);
  }
}
__device__ __forceinline__ void param_store(void* p, int bf16, int64_t c, float v) {
  if (bf16)
    static_cast<__nv_bfloat16*>(p)[c] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(p)[c] = v;
}

struct FwdArgs {
  const void* x;
  const void* gamma;
  const void* beta;
  void* y;
  float* mean;
  float* rstd;
  int64_t rows, xs, ys, chunk;  // chunk: rows per block
  int cols, param_bf16, param_vec, groups, period, classes;
  float eps, inv_cols;
  int* err;
  int cl;  // blocks per row, where a cluster shares it
};

struct BwdArgs {
  const void* dout;
  const void* x;
  const float* mean;
  const float* rstd;
  const void* gamma;
  void* dx;
  float* partial;  // [2][groups][cols]: the scale's sums, then the shift's; null without weight gradients
  int64_t rows, dos, xs, dxs, chunk;  // chunk: rows per block
  int cols, param_bf16, param_vec, groups, period, classes;
  float inv_cols;
  int* err;
  int cl;  // blocks per row, where a cluster shares it
};

// Sum over the TPR threads of a row.  Up to a warp: shuffles; of two sums, the halves of the row's lanes take one each
// after the first step.  More: each warp leaves its sums in one of two buffers that alternate from row to row, so one
// barrier of the row's own threads is enough (a buffer is written again only after the barrier of the row between).
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int slot, int& phase) {
  static_assert(N <= 2 && TPR >= 4, "one or two sums");
  constexpr int W = TPR < 32 ? TPR : 32, NW = TPR / 32;
  const bool up = N == 2 && (threadIdx.x & (W / 2));
  float s = up ? v[N - 1] : v[0];
  s += __shfl_xor_sync(0xffffffffu, N == 1 || up ? v[0] : v[N - 1], W / 2);
#pragma unroll
  for (int o = W / 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if constexpr (TPR <= 32) {
    if constexpr (N == 2) {
      const float other = __shfl_xor_sync(0xffffffffu, s, W / 2);
      v[0] = up ? other : s;
      v[1] = up ? s : other;
    } else {
      v[0] = s;
    }
  } else {
    float* buf = red + (slot * 2 + phase) * NW * N;
    phase ^= 1;
    const int w = (threadIdx.x % TPR) >> 5, lane = threadIdx.x & 31;
    if (lane % (W / N) == 0) buf[w * N + up] = s;
    asm volatile("bar.sync %0, %1;" ::"r"(slot + 1), "n"(TPR) : "memory");
    if constexpr (N == 2) {
      uint64_t a = 0, b = 0;  // a pair of zeros
#pragma unroll
      for (int i = 0; i < NW; i += 2) {
        const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(buf + i * N);
        a = f2_add(a, q.x), b = f2_add(b, q.y);
      }
      f2_unpack(f2_add(a, b), v[0], v[N - 1]);
    } else {
      uint64_t a = 0;
#pragma unroll
      for (int i = 0; i < NW; i += 2) a = f2_add(a, *reinterpret_cast<const uint64_t*>(buf + i));
      float lo, hi;
      f2_unpack(a, lo, hi);
      v[0] = lo + hi;
    }
  }
}

// ... and over the blocks (cl of them) of a cluster that share a row: every warp sends its sums to every block, whose mbarrier counts
// their bytes, and each thread adds up what arrived.  Buffers and mbarriers alternate: one is filled again only after
// every warp has sent its sums of the time between, which it does after reading this one.  (A block's barrier and then
// the cluster's took 0.9 us of the 2.0 that a row of the gradients took.)
constexpr int kMaxCluster = 8;

template <int NW, int N>
struct ClusterSums {
  float sums[2][kMaxCluster * NW * N];  // of [block][warp]
  uint64_t ready[2];
  int abort;

  __device__ __forceinline__ void init() {
    if (threadIdx.x == 0) {
      mbar_init(&ready[0], 1);
      mbar_init(&ready[1], 1);
      abort = 0;
      fence_barrier_init();
    }
    cluster_sync_all();  // every block of the cluster is there, its mbarriers too
  }
  // A warp's sums: of two, the lower half of the lanes gets the first, the upper half the second.
  static __device__ __forceinline__ float warp_sum(float x, float y, bool up) {
    float s = up ? y : x;
    s += __shfl_xor_sync(0xffffffffu, N == 1 || up ? x : y, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  }
  // n: the number of the call.  False, of whole warps, when the others' sums do not come.
  __device__ __forceinline__ bool sum(float (&v)[N], int rank, int cl, uint32_t n, int* err) {
    const uint32_t ph = n & 1;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const bool up = N == 2 && (lane & 16);
    if (threadIdx.x == 0) mbar_expect_tx(&ready[ph], cl * NW * N * 4);
    float s = warp_sum(v[0], v[N - 1], up);
    const int to = lane % (32 / N);
    if (to < cl) {
      const uint32_t dst = mapa_shared(smem_u32(&sums[ph][(rank * NW + w) * N + up]), to);
      const uint32_t bar = mapa_shared(smem_u32(&ready[ph]), to);
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(dst),
                   "r"(__float_as_uint(s)), "r"(bar)
                   : "memory");
    }
    const bool ok = mbar_wait_cluster(&ready[ph], (n >> 1) & 1, &abort, err);
    if (!__all_sync(0xffffffffu, ok)) return false;
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int i = lane; i < kMaxCluster * NW; i += 32)
      if (i < cl * NW) x += sums[ph][i * N], y += sums[ph][i * N + N - 1];
    s = warp_sum(x, y, up);
    if constexpr (N == 2) {
      const float other = __shfl_xor_sync(0xffffffffu, s, 16);
      v[0] = up ? other : s;
      v[1] = up ? s : other;
    } else {
      v[0] = s;
    }
    return true;
  }
};

// The N elements that a thread holds of a row as N / 2 pairs, so that the arithmetic
// runs on two elements per instruction (with scalar arithmetic both directions were
// bound by instructions, not by memory: 33 per element in the backward pass).
template <typename T, int VEC, int NV>
__device__ __forceinline__ void unpack(const Pack<T, VEC> (&raw)[NV], uint64_t (&v)[NV * VEC / 2]) {
#pragma unroll
  for (int e = 0; e < NV * VEC; e += 2)
    v[e / 2] = f2_pack(to_f32(raw[e / VEC].v[e % VEC]), to_f32(raw[(e + 1) / VEC].v[(e + 1) % VEC]));
}
template <int VEC, int NV>
__device__ __forceinline__ void unpack(const Pack<__nv_bfloat16, VEC> (&raw)[NV], uint64_t (&v)[NV * VEC / 2]) {
  if constexpr (VEC == 1) {
#pragma unroll
    for (int i = 0; i < NV; i += 2) v[i / 2] = f2_pack(to_f32(raw[i].v[0]), to_f32(raw[i + 1].v[0]));
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[i]);
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j)  // a bf16 is the upper half of its f32
        v[i * VEC / 2 + j] = f2_pack(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
    }
  }
}
// Where a ragged row begins and ends within its 16-byte vectors: `shift` elements of the first one lie before the row,
// `tail` elements of the last one (its number `tail_i` of thread `tail_l`) are the row's.  All alike for the rows of a
// block, so what is done about them branches with the block; only two threads of a row hold such vectors.
template <int VEC>
struct Edges {
  int shift, tail;
  bool head;    // this thread's first vector begins before the row
  int tail_at;  // the number of this thread's vector that the row ends in (-1: none, or at its end)
  uint32_t keep[VEC >= 4 ? 4 : 1];  // the first vector's bits that are the row's
};

template <typename T, int VEC, int NV, int TPR>
__device__ __forceinline__ Edges<VEC> find_edges(int shift, int cols, int l, int rank) {
  Edges<VEC> e;
  const int last = (cols + shift - 1) / VEC, mine = rank * NV * TPR + l;  // vectors of the row, of this thread
  e.shift = shift;
  e.tail = cols + shift - last * VEC;
  e.head = mine == 0 && shift > 0;
  e.tail_at = e.tail < VEC && last >= mine && (last - mine) % TPR == 0 && (last - mine) / TPR < NV ? (last - mine) / TPR : -1;
  constexpr int per = 4 / sizeof(T);  // elements per word
#pragma unroll
  for (int w = 0; w < 4 && VEC >= 4; ++w) {
    const int dead = shift - w * per;  // of this word's elements
    e.keep[w] = !e.head || dead <= 0 ? ~0u : dead >= per ? 0u : 0xffff0000u;
  }
  return e;
}

// The part of an edge vector that is the row's, in as few aligned stores as it has binary digits.
template <typename T, int VEC>
__device__ __forceinline__ void store_edge(T* at, const Pack<T, VEC>& o, bool head, bool tail, const Edges<VEC>& e) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&o);
  if (head && tail) {  // a row within one vector
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (j >= e.shift && j < e.tail) at[j] = o.v[j];
  } else if (sizeof(T) == 4) {
    if (head) {
      if (e.shift & 1) at[e.shift] = e.shift == 1 ? o.v[1] : o.v[VEC - 1];
      if (e.shift <= 2) *reinterpret_cast<uint2*>(at + 2) = make_uint2(w[2], w[3]);
    } else {
      if (e.tail >= 2) *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
      if (e.tail & 1) at[e.tail - 1] = e.tail == 1 ? o.v[0] : o.v[2 % VEC];
    }
  } else {
    uint32_t* at32 = reinterpret_cast<uint32_t*>(at);
    if (head) {
      const int odd = e.shift >> 1, first = (e.shift + 1) >> 1;  // the half dead word, the first word that lives
      const uint32_t half = odd == 0 ? w[0] : odd == 1 ? w[1] : odd == 2 ? w[2] : w[3];
      if (e.shift & 1) reinterpret_cast<uint16_t*>(at)[e.shift] = (uint16_t)(half >> 16);
      if (first == 1) at32[1] = w[1];
      if (first == 3) at32[3] = w[3];
      if (first <= 2) *reinterpret_cast<uint2*>(at32 + 2) = make_uint2(w[2], w[3]);
    } else {
      const int odd = e.tail >> 1;
      const uint32_t half = odd == 0 ? w[0] : odd == 1 ? w[1] : odd == 2 ? w[2] : w[3];
      if (e.tail >= 4) *reinterpret_cast<uint2*>(at32) = make_uint2(w[0], w[1]);
      if (e.tail & 2) at32[e.tail >= 4 ? 2 : 0] = e.tail >= 4 ? w[2] : w[0];
      if (e.tail & 1) reinterpret_cast<uint16_t*>(at)[e.tail - 1] = (uint16_t)half;
    }
  }
}

// first: the column of the thread's first element; the vectors lie `step` columns apart.
template <typename T, int VEC, int NV, bool RAG>
__device__ __forceinline__ void store_pairs(T* row, int first, int step, int cols, const uint64_t (&v)[NV * VEC / 2],
                                            const Edges<VEC>& edges) {
  Pack<T, VEC> o[NV];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < NV * VEC; e += 2)
      f2_unpack(v[e / 2], o[e / VEC].v[e % VEC], o[(e + 1) / VEC].v[(e + 1) % VEC]);
  } else {
#pragma unroll
    for (int e = 0; e < NV * VEC; e += 2) {
      float lo, hi;
      f2_unpack(v[e / 2], lo, hi);
      const uint32_t w = pack_bf16(lo, hi);
      if constexpr (VEC > 1) {
        reinterpret_cast<uint32_t*>(&o[e / VEC])[e % VEC / 2] = w;
      } else {
        o[e].v[0] = __ushort_as_bfloat16((unsigned short)w);
        o[e + 1].v[0] = __ushort_as_bfloat16((unsigned short)(w >> 16));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + i * step;
    if constexpr (RAG) {
      const bool head = i == 0 && edges.head, tail = i == edges.tail_at;
      if (head || tail) store_edge<T, VEC>(row + c, o[i], head, tail, edges);
      else if (c < cols) *reinterpret_cast<Pack<T, VEC>*>(row + c) = o[i];
    } else {
      if (c < cols) *reinterpret_cast<Pack<T, VEC>*>(row + c) = o[i];
    }
  }
}
template <int VEC, int NV, bool RAG>
__device__ __forceinline__ void load_params(const void* p, int bf16, int vec, int first, int step, int cols, float other,
                                            uint64_t (&v)[NV * VEC / 2]) {
  float f[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + i * step;
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[i][j] = other;
    if (!p) continue;
    if constexpr (RAG) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (c + j >= 0 && c + j < cols) f[i][j] = param_at(p, bf16, c + j);
    } else {
      if (c < cols) params_at<VEC>(p, bf16, vec, c, f[i]);
    }
  }
#pragma unroll
  for (int e = 0; e < NV * VEC; e += 2) v[e / 2] = f2_pack(f[e / VEC][e % VEC], f[(e + 1) / VEC][(e + 1) % VEC]);
}
__device__ __forceinline__ float f2_total(uint64_t v) {
  float lo, hi;
  f2_unpack(v, lo, hi);
  return lo + hi;
}

// Each thread copies its own elements of the rows to come into its own slots of
// shared memory (cp.async) and reads them back itself: loads STAGES rows ahead
// without registers and without barriers.  Of a copy, the first n bytes are read and
// the rest is filled with 0: elements past the end of a row, and rows past the end.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int n) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The rows of a block's run, slot by slot (RPB rows at a time), of NT tensors.
//
// RAG: rows whose length or distance is no multiple of a 16-byte access.  All rows
// `period` apart start equally far (`shift` elements) behind a 16-byte boundary, and a
// block takes rows of one such class only: its threads own aligned vectors, the first
// one beginning `shift` elements before the row, and the columns of a thread stay the
// same from row to row.  (Element by element, 32768 rows of 1001 bf16 took 76 us in
// the backward pass, and this way 50.)
template <typename T, int VEC, int NV, int TPR, int BT, int STAGES, int NT, bool RAG>
struct Rows {
  // cp.async moves 4 bytes at least; smaller elements come one row ahead through registers
  static constexpr bool kAsync = sizeof(T) * VEC >= 4;
  static constexpr int RPB = BT / TPR;
  static constexpr int kBytes = kAsync ? BT * STAGES * NT * NV * VEC * (int)sizeof(T) : 0;
  using P = Pack<T, VEC>;
  P* slots;  // [STAGES][NT][NV][BT]
  const T* base[NT];
  const T* src[NT];  // this thread's first element in the row that is fetched next
  int64_t step[NT], ahead, last;
  int first_col, cols, head, tail;
  P reg[NT][NV];

  __device__ __forceinline__ void init(int n, const void* p, int64_t stride, int64_t row, int period) {
    base[n] = static_cast<const T*>(p);
    src[n] = base[n] + row * stride + first_col;
    step[n] = RPB * period * stride;
  }
  // `at` and `end` count rows of the block's class
  __device__ __forceinline__ void start(void* smem, int64_t at, int64_t end) {
    slots = static_cast<P*>(smem);
    ahead = at, last = end;
    head = tail = 0;
#pragma unroll
    for (int i = 0; i < (kAsync ? STAGES - 1 : 1); ++i) fetch();
  }
  __device__ __forceinline__ void fetch() {
    const bool in = ahead < last;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = first_col + i * TPR * VEC;
        const bool read = in && c < cols;
        const T* s = read ? src[n] + i * TPR * VEC : base[n];
        if constexpr (kAsync) {
          const int count = !read ? 0 : RAG ? min(VEC, cols - c) : VEC;
          copy_async<sizeof(P)>(smem_u32(slots + ((head * NT + n) * NV + i) * BT + threadIdx.x), s, count * (int)sizeof(T));
        } else {
          reg[n][i] = {};
          if (read) reg[n][i] = *reinterpret_cast<const P*>(s);
        }
      }
      src[n] += step[n];
    }
    if constexpr (kAsync) copy_commit();
    head = head + 1 == STAGES ? 0 : head + 1;
    ahead += RPB;
  }
  // The oldest row's elements as f32 pairs (0 outside the row), and the next fetch.  A slot is filled again a row
  // after it was read.
  __device__ __forceinline__ void take(uint64_t (&v)[NT][NV * VEC / 2], const Edges<VEC>& edges) {
    if constexpr (kAsync) copy_wait<STAGES - 2>();
    P c[NT][NV];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < NV; ++i) c[n][i] = kAsync ? slots[((tail * NT + n) * NV + i) * BT + threadIdx.x] : reg[n][i];
    tail = tail + 1 == STAGES ? 0 : tail + 1;
    if constexpr (RAG) {  // without the end of the row before
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int w = 0; w < 4; ++w) reinterpret_cast<uint32_t*>(&c[n][0])[w] &= edges.keep[w];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) unpack(c[n], v[n]);
    fetch();
  }
  __device__ __forceinline__ void drain() {
    if constexpr (kAsync) copy_wait<0>();
  }
};

// A block's rows: the rows r = cls + period * j, j in [first, last).
struct Run {
  int cls, period;
  int64_t first, last;
  __device__ __forceinline__ Run(int64_t rows, int period_, int classes, int64_t chunk, int block) : period(period_) {
    cls = block % classes;
    first = block / classes * chunk;
    last = min((rows - cls + period - 1) / period, first + chunk);
  }
  __device__ __forceinline__ int64_t row(int64_t j) const { return cls + period * j; }
};

// How many elements row `cls` starts behind a 16-byte boundary.
template <typename T, bool RAG>
__device__ __forceinline__ int row_shift(const void* p, int64_t stride, int cls) {
  if constexpr (!RAG) return 0;
  return (int)((reinterpret_cast<uintptr_t>(p) / sizeof(T) + cls * stride) % (16 / sizeof(T)));
}

// ---------------------------------------------------------------- forward
// A block takes a run of rows; scale and shift stay in registers.  CL blocks share longer rows.
template <typename T, int VEC, int NV, int TPR, int BT, int STAGES, bool RAG, bool CL>
__global__ void __launch_bounds__(BT, 512 / BT) layernorm_fwd_kernel(const FwdArgs p) {
  constexpr int RPB = BT / TPR, NW = TPR > 32 ? TPR / 32 : 1, N2 = NV * VEC / 2;
  __shared__ __align__(16) float red[CL ? 4 : RPB * 2 * NW];
  __shared__ __align__(16) ClusterSums<NW, 1> cluster;
  extern __shared__ __align__(16) uint8_t dyn[];
  const int slot = threadIdx.x / TPR, l = threadIdx.x % TPR, rank = CL ? (int)cluster_rank() : 0, cl = CL ? p.cl : 1;
  const Run run(p.rows, p.period, p.classes, p.chunk, blockIdx.x / cl);
  const int shift = row_shift<T, RAG>(p.x, p.xs, run.cls), first_col = (rank * NV * TPR + l) * VEC - shift;
  const Edges<VEC> edges = find_edges<T, VEC, NV, TPR>(shift, p.cols, l, rank);
  static_assert(!CL || RPB == 1, "one row per cluster");
  if constexpr (CL) cluster.init();
  Rows<T, VEC, NV, TPR, BT, STAGES, 1, RAG> rows;
  rows.first_col = first_col;
  rows.cols = p.cols;
  rows.init(0, p.x, p.xs, run.row(run.first + slot), run.period);
  rows.start(dyn, run.first + slot, run.last);
  uint64_t g[N2], b[N2];
  load_params<VEC, NV, RAG>(p.gamma, p.param_bf16, p.param_vec, first_col, TPR * VEC, p.cols, 1.f, g);
  load_params<VEC, NV, RAG>(p.beta, p.param_bf16, p.param_vec, first_col, TPR * VEC, p.cols, 0.f, b);
  int phase = 0;
  uint32_t sum_number = 0;
  for (int64_t j0 = run.first; j0 < run.last; j0 += RPB) {
    if (TPR >= 32 && j0 + slot >= run.last) break;  // whole warps (and whole barrier groups) leave together
    uint64_t v[1][N2];
    rows.take(v, edges);
    uint64_t a = f2_pack(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < N2; ++e) a = f2_add(a, v[0][e]);
    float s[1] = {f2_total(a)};
    if constexpr (!CL) row_sum<TPR, 1>(s, red, slot, phase);
    else if (!cluster.sum(s, rank, cl, sum_number++, p.err)) break;
    const float mean = s[0] * p.inv_cols;
    const uint64_t m2 = f2_pack(mean, mean);
    a = f2_pack(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < N2; ++e) v[0][e] = f2_sub(v[0][e], m2);
    // elements outside the row hold 0 - mean and must not count
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = first_col + i * TPR * VEC;
      if constexpr (VEC == 1) {
        if (i % 2 == 0) {
          float lo, hi;
          f2_unpack(v[0][i / 2], lo, hi);
          const uint64_t d = f2_pack(c < p.cols ? lo : 0.f, c + TPR < p.cols ? hi : 0.f);
          a = f2_fma(d, d, a);
        }
      } else {
        uint64_t q = f2_pack(0.f, 0.f);
        if (RAG && ((i == 0 && edges.head) || i == edges.tail_at)) {
          const int from = i == 0 && edges.head ? edges.shift : 0, to = i == edges.tail_at ? edges.tail : VEC;
#pragma unroll
          for (int j = 0; j < VEC; j += 2) {
            float lo, hi;
            f2_unpack(v[0][(i * VEC + j) / 2], lo, hi);
            v[0][(i * VEC + j) / 2] = f2_pack(j >= from && j < to ? lo : 0.f, j + 1 >= from && j + 1 < to ? hi : 0.f);
          }
        }
#pragma unroll
        for (int j = i * VEC / 2; j < (i + 1) * VEC / 2; ++j) q = f2_fma(v[0][j], v[0][j], q);
        if (c < p.cols) a = f2_add(a, q);
      }
    }
    s[0] = f2_total(a);
    if constexpr (!CL) row_sum<TPR, 1>(s, red, slot, phase);
    else if (!cluster.sum(s, rank, cl, sum_number++, p.err)) break;
    const float rstd = 1.0f / sqrtf(s[0] * p.inv_cols + p.eps);
    if (j0 + slot < run.last) {
      const int64_t row = run.row(j0 + slot);
      if (l == 0 && rank == 0) {
        if (p.mean) p.mean[row] = mean;
        if (p.rstd) p.rstd[row] = rstd;
      }
      const uint64_t r2 = f2_pack(rstd, rstd);
#pragma unroll
      for (int e = 0; e < N2; ++e) v[0][e] = f2_fma(f2_mul(v[0][e], r2), g[e], b[e]);
      store_pairs<T, VEC, NV, RAG>(static_cast<T*>(p.y) + row * p.ys, first_col, TPR * VEC, p.cols, v[0], edges);
    }
  }
  rows.drain();
  if constexpr (CL) cluster_sync_all();  // no sums on their way to a block that is gone
}

// Rows too long for registers: one block per row, re-read in each of three passes.
constexpr int kLoopThreads = 512;

__device__ __forceinline__ float2 block_sum2(float a, float b, float2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();  // red may still be read by the previous sum
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kLoopThreads / 32; ++i) {
    s.x += red[i].x;
    s.y += red[i].y;
  }
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kLoopThreads) layernorm_fwd_loop_kernel(const FwdArgs p) {
  __shared__ float2 red[kLoopThreads / 32];
  const int64_t row = blockIdx.x;
  const T* xr = static_cast<const T*>(p.x) + row * p.xs;
  T* yr = static_cast<T*>(p.y) + row * p.ys;
  float s = 0.f;
  for (int c = threadIdx.x; c < p.cols; c += kLoopThreads) s += to_f32(xr[c]);
  const float mean = block_sum2(s, 0.f, red).x * p.inv_cols;
  s = 0.f;
  for (int c = threadIdx.x; c < p.cols; c += kLoopThreads) {
    const float d = to_f32(xr[c]) - mean;
    s = fmaf(d, d, s);
  }
  const float rstd = 1.0f / sqrtf(block_sum2(s, 0.f, red).x * p.inv_cols + p.eps);
  if (threadIdx.x == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
  for (int c = threadIdx.x; c < p.cols; c += kLoopThreads) {
    const float g = p.gamma ? param_at(p.gamma, p.param_bf16, c) : 1.f;
    const float b = p.beta ? param_at(p.beta, p.param_bf16, c) : 0.f;
    from_f32(yr[c], fmaf((to_f32(xr[c]) - mean) * rstd, g, b));
  }
}

// --------------------------------------------------------------- backward
// Bytes of dynamic shared memory: the slots, or the columns' sums at the end.
template <typename T, int VEC, int NV, int TPR, int BT, int STAGES, bool RAG>
constexpr int bwd_smem() {
  const int slots = Rows<T, VEC, NV, TPR, BT, STAGES, 2, RAG>::kBytes;
  const int sums = BT * NV * VEC * (int)sizeof(float);
  return slots > sums ? slots : sums;
}

// A block takes a run of rows and keeps, per thread, the sums of dy z and dy over its
// rows for the columns that the thread owns; the row slots of the block are added in
// shared memory at the end, one partial row per block.  CL blocks share longer rows.
template <typename T, int VEC, int NV, int TPR, int BT, int STAGES, bool RAG, bool CL>
__global__ void __launch_bounds__(BT, (NV * VEC < 16 ? 768 : 512) / BT) layernorm_bwd_kernel(const BwdArgs p) {
  constexpr int RPB = BT / TPR, NW = TPR > 32 ? TPR / 32 : 1, N2 = NV * VEC / 2;
  __shared__ __align__(16) float red[CL ? 4 : RPB * 2 * NW * 2];
  __shared__ __align__(16) ClusterSums<NW, 2> cluster;
  extern __shared__ __align__(16) uint8_t dyn[];
  const int slot = threadIdx.x / TPR, l = threadIdx.x % TPR, rank = CL ? (int)cluster_rank() : 0, cl = CL ? p.cl : 1;
  const Run run(p.rows, p.period, p.classes, p.chunk, blockIdx.x / cl);
  const int shift = row_shift<T, RAG>(p.x, p.xs, run.cls), first_col = (rank * NV * TPR + l) * VEC - shift;
  const Edges<VEC> edges = find_edges<T, VEC, NV, TPR>(shift, p.cols, l, rank);
  static_assert(!CL || RPB == 1, "one row per cluster");
  if constexpr (CL) cluster.init();
  Rows<T, VEC, NV, TPR, BT, STAGES, 2, RAG> rows;
  rows.first_col = first_col;
  rows.cols = p.cols;
  rows.init(0, p.x, p.xs, run.row(run.first + slot), run.period);
  rows.init(1, p.dout, p.dos, run.row(run.first + slot), run.period);
  rows.start(dyn, run.first + slot, run.last);
  uint64_t ag[N2], ab[N2], g[N2];
  const uint64_t zero2 = f2_pack(0.f, 0.f);
#pragma unroll
  for (int e = 0; e < N2; ++e) ag[e] = ab[e] = zero2;
  load_params<VEC, NV, RAG>(p.gamma, p.param_bf16, p.param_vec, first_col, TPR * VEC, p.cols, 1.f, g);
  // the statistics of this row slot's next W rows, one row per lane, and of the W rows after
  constexpr int W = TPR < 32 ? TPR : 32;
  const int lane = l % W;
  auto stat = [&](const float* s, int64_t j) {
    j += slot + lane * RPB;
    return j < run.last ? s[run.row(j)] : 0.f;
  };
  float mean_w = stat(p.mean, run.first), rstd_w = stat(p.rstd, run.first);
  float mean_n = stat(p.mean, run.first + W * RPB), rstd_n = stat(p.rstd, run.first + W * RPB);
  int phase = 0, it = 0;
  uint32_t row_number = 0;
  for (int64_t j0 = run.first; j0 < run.last; j0 += RPB, ++it) {
    if (TPR >= 32 && j0 + slot >= run.last) break;
    if (it == W) {
      it = 0;
      mean_w = mean_n, rstd_w = rstd_n;
      mean_n = stat(p.mean, j0 + W * RPB), rstd_n = stat(p.rstd, j0 + W * RPB);
    }
    const float mean = __shfl_sync(0xffffffffu, mean_w, it, W), rstd = __shfl_sync(0xffffffffu, rstd_w, it, W);
    uint64_t v[2][N2];
    rows.take(v, edges);
    auto &z = v[0], &dz = v[1];
    // the difference first, as in the forward: as x rstd - mean rstd, z would be off by up to 2^-24 |mean| rstd
    const uint64_t r2 = f2_pack(rstd, rstd), m2 = f2_pack(mean, mean);
    uint64_t s0 = zero2, s1 = zero2;
#pragma unroll
    for (int e = 0; e < N2; ++e) {
      z[e] = f2_mul(f2_sub(z[e], m2), r2);
      ab[e] = f2_add(ab[e], dz[e]);
      ag[e] = f2_fma(dz[e], z[e], ag[e]);
      dz[e] = f2_mul(dz[e], g[e]);
      s0 = f2_add(s0, dz[e]);
      s1 = f2_fma(dz[e], z[e], s1);
    }
    float s[2] = {f2_total(s0), f2_total(s1)};
    if constexpr (!CL) row_sum<TPR, 2>(s, red, slot, phase);
    else if (!cluster.sum(s, rank, cl, row_number++, p.err)) break;
    const float k0 = -s[0] * p.inv_cols * rstd, k1 = -s[1] * p.inv_cols * rstd;
    const uint64_t k02 = f2_pack(k0, k0), k12 = f2_pack(k1, k1);
#pragma unroll
    for (int e = 0; e < N2; ++e) dz[e] = f2_fma(z[e], k12, f2_fma(dz[e], r2, k02));
    if (j0 + slot < run.last)
      store_pairs<T, VEC, NV, RAG>(static_cast<T*>(p.dx) + run.row(j0 + slot) * p.dxs, first_col, TPR * VEC, p.cols, dz,
                                   edges);
  }
  rows.drain();
  if constexpr (CL) cluster_sync_all();  // no sums on their way to a block that is gone
  if (!p.partial) return;
  const int64_t half = (int64_t)p.groups * p.cols;
  float* out = p.partial + (int64_t)(blockIdx.x / cl) * p.cols;
  // Through shared memory, so that a warp writes whole lines (a thread's own columns, stored from its registers, cost
  // 8 us per call at 16384 columns); a thread's vectors lie there as they do in the row.
  constexpr int WIDTH = TPR * NV * VEC;
  float* columns = reinterpret_cast<float*>(dyn);  // [RPB][WIDTH]
  const int first = rank * WIDTH - shift;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float f[NV * VEC];
#pragma unroll
    for (int e = 0; e < N2; ++e) f2_unpack(which ? ab[e] : ag[e], f[2 * e], f[2 * e + 1]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float* at = columns + slot * WIDTH + (i * TPR + l) * VEC;
      if constexpr (VEC == 1) {
        *at = f[i];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 4)
          *reinterpret_cast<float4*>(at + j) = make_float4(f[i * VEC + j], f[i * VEC + j + 1], f[i * VEC + j + 2], f[i * VEC + j + 3]);
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < WIDTH; e += BT) {
      const int c = first + e;
      if (c < 0 || c >= p.cols) continue;
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < RPB; ++r) s += columns[r * WIDTH + e];
      out[which * half + c] = s;
    }
  }
}

// Rows too long for registers: dx by one block per row (the row read twice), and
// the weight gradients by blocks that walk a slice of the rows, a column per thread.
template <typename T>
__global__ void __launch_bounds__(kLoopThreads) layernorm_bwd_loop_kernel(const BwdArgs p) {
  __shared__ float2 red[kLoopThreads / 32];
  const int64_t row = blockIdx.x;
  const T* xr = static_cast<const T*>(p.x) + row * p.xs;
  const T* dr = static_cast<const T*>(p.dout) + row * p.dos;
  T* wr = static_cast<T*>(p.dx) + row * p.dxs;
  const float mean = p.mean[row], rstd = p.rstd[row];
  float a = 0.f, b = 0.f;
  for (int c = threadIdx.x; c < p.cols; c += kLoopThreads) {
    const float dz = to_f32(dr[c]) * (p.gamma ? param_at(p.gamma, p.param_bf16, c) : 1.f);
    a += dz;
    b = fmaf(dz, (to_f32(xr[c]) - mean) * rstd, b);
  }
  const float2 s = block_sum2(a, b, red);
  const float m0 = s.x * p.inv_cols, m1 = s.y * p.inv_cols;
  for (int c = threadIdx.x; c < p.cols; c += kLoopThreads) {
    const float dz = to_f32(dr[c]) * (p.gamma ? param_at(p.gamma, p.param_bf16, c) : 1.f);
    from_f32(wr[c], rstd * (dz - m0 - (to_f32(xr[c]) - mean) * rstd * m1));
  }
}

constexpr int kColThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kColThreads) layernorm_bwd_columns_kernel(const BwdArgs p) {
  const int c = blockIdx.x * kColThreads + threadIdx.x;
  if (c >= p.cols) return;
  float g = 0.f, b = 0.f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float dy = to_f32(static_cast<const T*>(p.dout)[row * p.dos + c]);
    const float x = to_f32(static_cast<const T*>(p.x)[row * p.xs + c]);
    b += dy;
    g = fmaf(dy, (x - p.mean[row]) * p.rstd[row], g);
  }
  p.partial[(int64_t)blockIdx.y * p.cols + c] = g;
  p.partial[((int64_t)p.groups + blockIdx.y) * p.cols + c] = b;
}

// The partial rows of all blocks, added in a fixed order: a block takes 32 columns of one of the two gradients, its warps
// a share of the partial rows each, eight loads in flight (one after another, 300 rows took longer than the pass before).
// 32 warps, or 8 where there are columns enough for every SM's threads all the same.
constexpr int kFinUnroll = 8;

template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
    layernorm_bwd_finish_kernel(const float* partial, int groups, int cols, void* dgamma, void* dbeta, int param_bf16) {
  __shared__ float s[WARPS][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  grid_dep_wait();
  const float* src = partial + (int64_t)blockIdx.y * groups * cols + c;
  float v = 0.f;
  if (c < cols) {
    int r = w;
    for (; r + (kFinUnroll - 1) * WARPS < groups; r += kFinUnroll * WARPS) {
      float q[kFinUnroll];
#pragma unroll
      for (int i = 0; i < kFinUnroll; ++i) q[i] = src[(int64_t)(r + i * WARPS) * cols];
#pragma unroll
      for (int i = 0; i < kFinUnroll; ++i) v += q[i];
    }
    for (; r < groups; r += WARPS) v += src[(int64_t)r * cols];
  }
  s[w][lane] = v;
  __syncthreads();
  // the block's sums turned: WARPS neighbouring threads add one column's shares
  const int col = threadIdx.x / WARPS, share = threadIdx.x % WARPS;
  v = s[share][col];
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (share == 0 && blockIdx.x * 32 + col < cols)
    param_store(blockIdx.y ? dbeta : dgamma, param_bf16, blockIdx.x * 32 + col, v);
}

// ------------------------------------------------------------------- host
bool aligned(const void* p, int64_t stride, int vec, int size) {
  return reinterpret_cast<uintptr_t>(p) % (uintptr_t)(vec * size) == 0 && stride % vec == 0;
}

bool typed(const void* p, int32_t dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == PDB_F32 ? 4 : 2) == 0; }

int param_vec(const void* g, const void* b) {
  return ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

constexpr int kMaxCols = 1 << 30;

int check(int64_t rows, int64_t cols, int32_t dtype, int32_t param_dtype) {
  if (rows < 0 || cols < 0) return set_error(PDB_ERR_SHAPE, "layernorm: negative size");
  if (rows > 0x7fffffffLL) return set_error(PDB_ERR_SHAPE, "layernorm: rows > 2^31-1");
  if (cols > kMaxCols) return set_error(PDB_ERR_SHAPE, "layernorm: cols > 2^30");
  if (dtype != PDB_F32 && dtype != PDB_BF16) return set_error(PDB_ERR_UNSUPPORTED, "layernorm: unknown dtype %d", dtype);
  if (param_dtype != PDB_F32 && param_dtype != dtype)
    return set_error(PDB_ERR_UNSUPPORTED, "layernorm: gamma / beta must be f32 or of the rows' type");
  return PDB_OK;
}

// A launch's shape: NV vectors of VEC elements per thread, TPR threads per row, BT per
// block; `blocks` of them per SM share the rows of every class in runs.
template <typename Args>
void share_rows(Args& p, int rpb, int64_t blocks) {
  p.classes = (int)std::min<int64_t>(p.period, p.rows);
  const int64_t each = (p.rows + p.period - 1) / p.period, sets = (each + rpb - 1) / rpb;
  const int64_t runs = std::max<int64_t>(1, blocks / p.classes);
  p.chunk = (sets + runs - 1) / runs * rpb;
  p.groups = (int)((each + p.chunk - 1) / p.chunk * p.classes);
}

int sms() {
  int dev = 0;
  cudaGetDevice(&dev);
  return sm_count(dev);
}

// The most blocks that share the rows of the backward pass.
int64_t bwd_groups(int64_t rows, int sms) { return std::max<int64_t>(8, std::min<int64_t>(rows + 8, 4 * sms)); }

template <typename T>
bool rag_fits(const void* a, int64_t as, const void* b, int64_t bs) {
  constexpr int V = 16 / sizeof(T);
  return reinterpret_cast<uintptr_t>(a) % 16 == reinterpret_cast<uintptr_t>(b) % 16 && (as - bs) % V == 0;
}
template <typename T>
int rag_period(int64_t stride) {
  int p = 16 / sizeof(T);
  while (p > 1 && stride * (p / 2) % (16 / (int)sizeof(T)) == 0) p /= 2;
  return p;
}

// p.groups clusters of CL blocks
template <typename Args>
int launch(void (*kernel)(Args), const Args& p, int threads, int smem, int cl, cudaStream_t s) {
  if (smem > 40 * 1024)  // with the static arrays, 48 KB would be passed
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))
      return cuda_status(e, "layernorm: smem attribute"), -1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.groups * cl));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cl;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = cl > 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p)) return cuda_status(e, "layernorm launch"), -1;
  return 1;
}

// Clusters of cl blocks that the device holds at once (less than its SMs suggest: a cluster's blocks share a GPC).
template <typename Args>
int cluster_places(void (*kernel)(Args), int threads, int smem, int cl, std::atomic<int> (&known)[16][kMaxCluster + 1]) {
  int dev = 0;
  cudaGetDevice(&dev);
  int n = dev < 16 ? known[dev][cl].load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(cl);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cl;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();  // the launch itself says what is wrong
    return 1;
  }
  if (dev < 16) known[dev][cl].store(n, std::memory_order_relaxed);
  return n;
}

// 1: launched, 0: the row is too long for this shape, -1: an error
template <typename T, int VEC, int NV, int TPR, int BT, int STAGES, bool RAG, bool CL = false>
int launch_fwd(FwdArgs& p, int blocks, cudaStream_t s) {
  const int need = p.cols + (RAG ? VEC - 1 : 0);
  p.cl = (need + TPR * NV * VEC - 1) / (TPR * NV * VEC);
  if (p.cl > (CL ? kMaxCluster : 1)) return 0;
  const auto kernel = layernorm_fwd_kernel<T, VEC, NV, TPR, BT, STAGES, RAG, CL>;
  constexpr int smem = Rows<T, VEC, NV, TPR, BT, STAGES, 1, RAG>::kBytes;
  int64_t places = (int64_t)blocks * sms();
  if constexpr (CL) {
    static std::atomic<int> known[16][kMaxCluster + 1];
    places = cluster_places(kernel, BT, smem, p.cl, known);
  }
  share_rows(p, BT / TPR, places);
  return launch(kernel, p, BT, smem, p.cl, s);
}

// 32 elements per thread in the forward (16 of f32), 256 threads per block and runs for 4 blocks per SM (two are resident
// at 126 registers, so the grid takes two waves); measured over 32 MiB elements of bf16 from a cold L2: 27 to 29 us at the
// powers of two from 128 to 8192 columns, a copy 26.6; 33 us at 64 columns, where half of four threads' vectors are empty,
// as a quarter are at 768 and 1536 (31 us) and three eighths at 5120 (35).  128 columns on eight threads, half of whose
// vectors would be empty, took 6 us more than on four.  Rows above 16384 columns (f32: 8192) go to clusters of as many
// blocks as they need: 1000 x 32768 bf16 39 us, where one block per row that reads it three times took 78.  Element by
// element (tensors whose rows lie differently against 16 bytes) a thread takes 8, or 16 of long rows.
template <typename T, int VEC, bool RAG>
int dispatch_fwd(FwdArgs& p, cudaStream_t s) {
  if constexpr (VEC == 1) {
    int r = launch_fwd<T, 1, 8, 32, 256, 3, false>(p, 4, s);
    if (!r) r = launch_fwd<T, 1, 8, 256, 256, 3, false>(p, 4, s);
    if (!r) r = launch_fwd<T, 1, 16, 512, 512, 2, false>(p, 2, s);
    return r;
  } else {
    constexpr int NV = (sizeof(T) == 2 ? 32 : 16) / VEC;
    int r = launch_fwd<T, VEC, NV, 4, 256, 3, RAG>(p, 4, s);
    if (!r) r = launch_fwd<T, VEC, NV, 8, 256, 3, RAG>(p, 4, s);
    if (!r) r = launch_fwd<T, VEC, NV, 16, 256, 3, RAG>(p, 4, s);
    if (!r) r = launch_fwd<T, VEC, NV, 32, 256, 3, RAG>(p, 4, s);
    if (!r) r = launch_fwd<T, VEC, NV, 64, 256, 3, RAG>(p, 4, s);
    if (!r) r = launch_fwd<T, VEC, NV, 128, 256, 3, RAG>(p, 4, s);
    if (!r) r = launch_fwd<T, VEC, NV, 256, 256, 3, RAG>(p, 4, s);
    if (!r) r = launch_fwd<T, VEC, NV, 512, 512, 2, RAG>(p, 2, s);
    if (!r) r = launch_fwd<T, VEC, NV, 256, 256, 3, RAG, true>(p, 4, s);
    return r;
  }
}

template <typename T>
int forward(FwdArgs& p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  int done;
  if (p.cols % V == 0 && aligned(p.x, p.xs, V, sizeof(T)) && aligned(p.y, p.ys, V, sizeof(T))) {
    done = dispatch_fwd<T, V, false>(p, s);
  } else if (rag_fits<T>(p.x, p.xs, p.y, p.ys)) {
    p.period = rag_period<T>(p.xs);
    done = dispatch_fwd<T, V, true>(p, s);
  } else {
    done = dispatch_fwd<T, 1, false>(p, s);
  }
  if (done < 0) return PDB_ERR_CUDA;
  if (!done) layernorm_fwd_loop_kernel<T><<<(unsigned)p.rows, kLoopThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "layernorm forward launch");
}

template <typename T, int VEC, int NV, int TPR, int BT, int STAGES, bool RAG, bool CL = false>
int launch_bwd(BwdArgs& p, int blocks, cudaStream_t s) {
  const int need = p.cols + (RAG ? VEC - 1 : 0);
  p.cl = (need + TPR * NV * VEC - 1) / (TPR * NV * VEC);
  if (p.cl > (CL ? kMaxCluster : 1)) return 0;
  const auto kernel = layernorm_bwd_kernel<T, VEC, NV, TPR, BT, STAGES, RAG, CL>;
  constexpr int smem = bwd_smem<T, VEC, NV, TPR, BT, STAGES, RAG>();
  int64_t places = (int64_t)blocks * sms();
  if constexpr (CL) {
    static std::atomic<int> known[16][kMaxCluster + 1];
    places = cluster_places(kernel, BT, smem, p.cl, known);
  }
  share_rows(p, BT / TPR, places);
  return launch(kernel, p, BT, smem, p.cl, s);
}

// 16 elements per thread, whose sums and scale fill its registers: 512 threads per SM, three rows ahead.  32 MiB
// elements of bf16 with the sums' join, from a cold L2: 43 us at the powers of two from 64 to 4096 columns (38 where calls
// follow one another), a copy of as many bytes 37; 45 us at 8192, where an SM has one row at a time, and at 768 and 1536,
// where a quarter of the vectors are empty; 55 at 5120 (three eighths).  Blocks of 512 threads on f32 keep two rows
// (three, 196 KB, leave the caches too little: 83 against 74 us at 8192 columns).  Rows above 8192 columns go to clusters
// of as many blocks of 256 threads as they need (50 us at 16384, 54 at 32768); at 4100 to 8192 columns a cluster of two
// is no faster than one block of 512.
template <typename T, int VEC, bool RAG>
int dispatch_bwd(BwdArgs& p, cudaStream_t s) {
  constexpr int S = sizeof(T) == 4 ? 2 : 3;
  if constexpr (VEC == 1) {
    int r = launch_bwd<T, 1, 4, 32, 256, 3, false>(p, 3, s);
    if (!r) r = launch_bwd<T, 1, 4, 256, 256, 3, false>(p, 3, s);
    if (!r) r = launch_bwd<T, 1, 16, 512, 512, S, false>(p, 1, s);
    return r;
  } else {
    constexpr int NV = 16 / VEC;
    int r = launch_bwd<T, VEC, NV, 4, 256, 3, RAG>(p, 2, s);
    if (!r) r = launch_bwd<T, VEC, NV, 8, 256, 3, RAG>(p, 2, s);
    if (!r) r = launch_bwd<T, VEC, NV, 16, 256, 3, RAG>(p, 2, s);
    if (!r) r = launch_bwd<T, VEC, NV, 32, 256, 3, RAG>(p, 2, s);
    if (!r) r = launch_bwd<T, VEC, NV, 64, 256, 3, RAG>(p, 2, s);
    if (!r) r = launch_bwd<T, VEC, NV, 128, 256, 3, RAG>(p, 2, s);
    if (!r) r = launch_bwd<T, VEC, NV, 256, 512, S, RAG>(p, 1, s);
    if (!r) r = launch_bwd<T, VEC, NV, 512, 512, S, RAG>(p, 1, s);
    if (!r) r = launch_bwd<T, VEC, NV, 256, 256, S, RAG, true>(p, 2, s);
    return r;
  }
}

template <typename T>
int backward(BwdArgs& p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  int done;
  if (p.cols % V == 0 && aligned(p.x, p.xs, V, sizeof(T)) && aligned(p.dout, p.dos, V, sizeof(T)) &&
      aligned(p.dx, p.dxs, V, sizeof(T))) {
    done = dispatch_bwd<T, V, false>(p, s);
  } else if (rag_fits<T>(p.x, p.xs, p.dout, p.dos) && rag_fits<T>(p.x, p.xs, p.dx, p.dxs)) {
    p.period = rag_period<T>(p.xs);
    done = dispatch_bwd<T, V, true>(p, s);
  } else {
    done = dispatch_bwd<T, 1, false>(p, s);
  }
  if (done < 0) return PDB_ERR_CUDA;
  if (!done) {
    p.groups = (int)std::min<int64_t>(p.rows, 4 * sms());
    if (p.partial)  // first: dx may lie where x or dout does
      layernorm_bwd_columns_kernel<T>
          <<<dim3((unsigned)((p.cols + kColThreads - 1) / kColThreads), (unsigned)p.groups), kColThreads, 0, s>>>(p);
    layernorm_bwd_loop_kernel<T><<<(unsigned)p.rows, kLoopThreads, 0, s>>>(p);
  }
  return cuda_status(cudaGetLastError(), "layernorm backward launch");
}

}  // namespace
}  // namespace pdb

using namespace pdb;

extern "C" int pdb_layernorm_fwd(const pdb_layernorm_fwd_desc* d, void* stream) {
  if (!d) return set_error(PDB_ERR_ARG, "null descriptor");
  if (int st = check(d->rows, d->cols, d->dtype, d->param_dtype)) return st;
  if (d->rows > 1 && (d->x_row_stride < d->cols || d->y_row_stride < d->cols))
    return set_error(PDB_ERR_SHAPE, "row stride smaller than cols");
  if (d->rows > 0 && d->cols == 0 && (d->mean || d->rstd))
    return set_error(PDB_ERR_SHAPE, "layernorm: rows without columns have no statistics");
  if (d->rows == 0 || d->cols == 0) return PDB_OK;
  if (!d->x || !d->y) return set_error(PDB_ERR_ARG, "null x / y");
  if (d->rows > 1 && d->y == d->x && d->y_row_stride != d->x_row_stride)
    return set_error(PDB_ERR_ARG, "layernorm: rows that are normed in place have one row stride");
  if (!typed(d->x, d->dtype) || !typed(d->y, d->dtype) || !typed(d->gamma, d->param_dtype) || !typed(d->beta, d->param_dtype))
    return set_error(PDB_ERR_ALIGN, "layernorm: a tensor is not aligned to its type");
  FwdArgs p{d->x, d->gamma, d->beta, d->y, d->mean, d->rstd, d->rows, d->x_row_stride, d->y_row_stride,
                  0, (int)d->cols, d->param_dtype == PDB_BF16, param_vec(d->gamma, d->beta), 0, 1, 1, (float)d->eps,
                  (float)(1.0 / (double)d->cols), device_error_flag()};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return d->dtype == PDB_F32 ? forward<float>(p, s) : forward<__nv_bfloat16>(p, s);
}

extern "C" size_t pdb_layernorm_bwd_workspace_size(const pdb_layernorm_bwd_desc* d) {
  if (!d || d->rows < 0 || d->cols <= 0 || d->cols > kMaxCols || !d->dgamma) return 0;
  return (size_t)2 * bwd_groups(d->rows, sms()) * d->cols * sizeof(float);
}

extern "C" int pdb_layernorm_bwd(const pdb_layernorm_bwd_desc* d, void* stream) {
  if (!d) return set_error(PDB_ERR_ARG, "null descriptor");
  if (int st = check(d->rows, d->cols, d->dtype, d->param_dtype)) return st;
  if (d->rows > 1 && (d->x_row_stride < d->cols || d->dout_row_stride < d->cols || d->dx_row_stride < d->cols))
    return set_error(PDB_ERR_SHAPE, "row stride smaller than cols");
  if (d->cols == 0) return PDB_OK;
  if ((d->dgamma == nullptr) != (d->dbeta == nullptr))
    return set_error(PDB_ERR_ARG, "dgamma and dbeta are computed together: give both or neither");
  if (d->rows > 0 && (!d->x || !d->dout || !d->dx || !d->mean || !d->rstd))
    return set_error(PDB_ERR_ARG, "null x / dout / dx / mean / rstd");
  if (d->rows > 1 && ((d->dx == d->x && d->dx_row_stride != d->x_row_stride) ||
                      (d->dx == d->dout && d->dx_row_stride != d->dout_row_stride)))
    return set_error(PDB_ERR_ARG, "layernorm backward: a gradient that is taken in place has its tensor's row stride");
  if (d->dgamma && (!d->workspace || d->workspace_bytes < pdb_layernorm_bwd_workspace_size(d)))
    return set_error(PDB_ERR_ARG, "layernorm backward: workspace too small");
  if (!typed(d->x, d->dtype) || !typed(d->dout, d->dtype) || !typed(d->dx, d->dtype) || !typed(d->gamma, d->param_dtype) ||
      !typed(d->dgamma, d->param_dtype) || !typed(d->dbeta, d->param_dtype) || !typed(d->workspace, PDB_F32))
    return set_error(PDB_ERR_ALIGN, "layernorm backward: a tensor is not aligned to its type");
  BwdArgs p{d->dout, d->x, d->mean, d->rstd, d->gamma, d->dx,
                  d->dgamma ? static_cast<float*>(d->workspace) : nullptr, d->rows, d->dout_row_stride,
                  d->x_row_stride, d->dx_row_stride, 0, (int)d->cols, d->param_dtype == PDB_BF16,
                  param_vec(d->gamma, nullptr), 0, 1, 1, (float)(1.0 / (double)d->cols), device_error_flag()};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->rows > 0)
    if (int st = d->dtype == PDB_F32 ? backward<float>(p, s) : backward<__nv_bfloat16>(p, s)) return st;
  if (!d->dgamma) return PDB_OK;
  // its blocks may be scheduled while the pass before drains; they wait for that pass's memory
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((d->cols + 31) / 32), 2);
  const bool wide = (int)cfg.gridDim.x > sms();
  cfg.blockDim = dim3(32 * (wide ? 8 : 32));
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, wide ? layernorm_bwd_finish_kernel<8> : layernorm_bwd_finish_kernel<32>,
                                        (const float*)p.partial, d->rows > 0 ? p.groups : 0, p.cols, d->dgamma, d->dbeta,
                                        p.param_bf16),
                     "layernorm backward finish launch");
}
