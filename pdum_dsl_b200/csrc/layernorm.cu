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
// keep it in registers between its two reductions.
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
  int64_t rows, xs, ys;
  int cols, param_bf16;
  float eps, inv_cols;
};

struct BwdArgs {
  const void* dout;
  const void* x;
  const float* mean;
  const float* rstd;
  const void* gamma;
  void* dx;
  float* partial;  // [2][groups][cols]: the scale's sums, then the shift's; null without weight gradients
  int64_t rows, dos, xs, dxs;
  int cols, param_bf16, groups;
  float inv_cols;
};

// Sum over the TPR threads of a row.  Up to a warp: shuffles.  More: each warp
// leaves its sum in one of two buffers that alternate from row to row, so one
// barrier of the row's own threads is enough (a buffer is written again only
// after the barrier of the row between).
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int slot, int& phase) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  if constexpr (TPR > 32) {
    constexpr int NW = TPR / 32;
    float* buf = red + (slot * 2 + phase) * NW * N;
    phase ^= 1;
    const int w = (threadIdx.x % TPR) >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) buf[w * N + n] = v[n];
    asm volatile("bar.sync %0, %1;" ::"r"(slot + 1), "n"(TPR) : "memory");
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) s += buf[i * N + n];
      v[n] = s;
    }
  }
}

// ---------------------------------------------------------------- forward
template <typename T, int VEC, int NV, int TPR, int BT>
__global__ void __launch_bounds__(BT) layernorm_fwd_kernel(const FwdArgs p) {
  constexpr int RPB = BT / TPR, NW = TPR > 32 ? TPR / 32 : 1;
  __shared__ float red[RPB * 2 * NW];
  const int slot = threadIdx.x / TPR, l = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + slot;
  if (TPR >= 32 && row >= p.rows) return;  // whole warps (and whole barrier groups) leave together
  const bool live = row < p.rows;
  const T* xr = static_cast<const T*>(p.x) + (live ? row : 0) * p.xs;
  T* yr = static_cast<T*>(p.y) + (live ? row : 0) * p.ys;
  Pack<T, VEC> raw[NV];
  float s[1] = {0.f};
  int phase = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (l + i * TPR) * VEC;
    if (c < p.cols) {
      raw[i] = *reinterpret_cast<const Pack<T, VEC>*>(xr + c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] += to_f32(raw[i].v[j]);
    }
  }
  row_sum<TPR, 1>(s, red, slot, phase);
  const float mean = s[0] * p.inv_cols;
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((l + i * TPR) * VEC < p.cols)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = to_f32(raw[i].v[j]) - mean;
        s[0] = fmaf(d, d, s[0]);
      }
  row_sum<TPR, 1>(s, red, slot, phase);
  const float rstd = 1.0f / sqrtf(s[0] * p.inv_cols + p.eps);
  if (!live) return;
  if (l == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (l + i * TPR) * VEC;
    if (c < p.cols) {
      Pack<T, VEC> o;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float g = p.gamma ? param_at(p.gamma, p.param_bf16, c + j) : 1.f;
        const float b = p.beta ? param_at(p.beta, p.param_bf16, c + j) : 0.f;
        from_f32(o.v[j], fmaf((to_f32(raw[i].v[j]) - mean) * rstd, g, b));
      }
      *reinterpret_cast<Pack<T, VEC>*>(yr + c) = o;
    }
  }
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
// A block takes rows at a stride of the grid and keeps, per thread, the sums of
// dy z and dy over its rows for the columns that the thread owns; the row slots
// of the block are added in shared memory at the end, one partial row per block.
template <typename T, int VEC, int NV, int TPR, int BT>
__global__ void __launch_bounds__(BT) layernorm_bwd_kernel(const BwdArgs p) {
  constexpr int RPB = BT / TPR, NW = TPR > 32 ? TPR / 32 : 1;
  __shared__ float red[RPB * 2 * NW * 2];
  extern __shared__ float cols_s[];  // [RPB][TPR * NV * VEC], when RPB > 1
  const int slot = threadIdx.x / TPR, l = threadIdx.x % TPR;
  float ag[NV][VEC], ab[NV][VEC], g[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = (l + i * TPR) * VEC + j;
      ag[i][j] = ab[i][j] = 0.f;
      g[i][j] = (p.gamma && c < p.cols) ? param_at(p.gamma, p.param_bf16, c) : 1.f;
    }
  int phase = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < p.rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + slot;
    if (TPR >= 32 && row >= p.rows) break;
    const bool live = row < p.rows;
    const int64_t rr = live ? row : 0;
    const T* xr = static_cast<const T*>(p.x) + rr * p.xs;
    const T* dr = static_cast<const T*>(p.dout) + rr * p.dos;
    T* wr = static_cast<T*>(p.dx) + rr * p.dxs;
    const float mean = p.mean[rr], rstd = p.rstd[rr];
    Pack<T, VEC> xv[NV], dv[NV];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (l + i * TPR) * VEC;
      if (live && c < p.cols) {
        xv[i] = *reinterpret_cast<const Pack<T, VEC>*>(xr + c);
        dv[i] = *reinterpret_cast<const Pack<T, VEC>*>(dr + c);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (live && (l + i * TPR) * VEC < p.cols)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float z = (to_f32(xv[i].v[j]) - mean) * rstd, dy = to_f32(dv[i].v[j]);
          const float dz = dy * g[i][j];
          s[0] += dz;
          s[1] = fmaf(dz, z, s[1]);
          ab[i][j] += dy;
          ag[i][j] = fmaf(dy, z, ag[i][j]);
        }
    }
    row_sum<TPR, 2>(s, red, slot, phase);
    const float m0 = s[0] * p.inv_cols, m1 = s[1] * p.inv_cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (l + i * TPR) * VEC;
      if (live && c < p.cols) {
        Pack<T, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float z = (to_f32(xv[i].v[j]) - mean) * rstd;
          from_f32(o.v[j], rstd * (fmaf(to_f32(dv[i].v[j]), g[i][j], -m0) - z * m1));
        }
        *reinterpret_cast<Pack<T, VEC>*>(wr + c) = o;
      }
    }
  }
  if (!p.partial) return;
  const int64_t half = (int64_t)p.groups * p.cols;
  float* out = p.partial + (int64_t)blockIdx.x * p.cols;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = (l + i * TPR) * VEC + j;
        if (c < p.cols) {
          out[c] = ag[i][j];
          out[half + c] = ab[i][j];
        }
      }
  } else {
    constexpr int WIDTH = TPR * NV * VEC;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          cols_s[slot * WIDTH + (l + i * TPR) * VEC + j] = which ? ab[i][j] : ag[i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < p.cols; c += BT) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < RPB; ++r) s += cols_s[r * WIDTH + c];
        out[which * half + c] = s;
      }
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

// The partial rows of all blocks, added in a fixed order: a warp takes 32 columns
// of one of the two gradients, 8 warps of a block share the partial rows.
constexpr int kFinWarps = 8;

__global__ void __launch_bounds__(32 * kFinWarps)
    layernorm_bwd_finish_kernel(const float* partial, int groups, int cols, void* dgamma, void* dbeta, int param_bf16) {
  __shared__ float s[kFinWarps][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const float* src = partial + (int64_t)blockIdx.y * groups * cols;
  float v = 0.f;
  if (c < cols)
    for (int r = w; r < groups; r += kFinWarps) v += src[(int64_t)r * cols + c];
  s[w][lane] = v;
  __syncthreads();
  if (w == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < kFinWarps; ++i) v += s[i][lane];
    param_store(blockIdx.y ? dbeta : dgamma, param_bf16, c, v);
  }
}

// ------------------------------------------------------------------- host
bool aligned(const void* p, int64_t stride, int vec, int size) {
  return reinterpret_cast<uintptr_t>(p) % (uintptr_t)(vec * size) == 0 && stride % vec == 0;
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

// The widths that a row's threads and registers give: VEC elements x NV vectors x
// TPR threads.  The smallest that holds the row is taken.
template <typename T, int VEC, int NV, int TPR, int BT>
void launch_fwd(const FwdArgs& p, cudaStream_t s) {
  const int64_t grid = (p.rows + BT / TPR - 1) / (BT / TPR);
  layernorm_fwd_kernel<T, VEC, NV, TPR, BT><<<(unsigned)grid, BT, 0, s>>>(p);
}

template <typename T, int VEC>
bool dispatch_fwd(const FwdArgs& p, cudaStream_t s) {
  const int64_t nv = ((int64_t)p.cols + VEC - 1) / VEC;
  if (nv <= 16) launch_fwd<T, VEC, 1, 16, 256>(p, s);
  else if (nv <= 32) launch_fwd<T, VEC, 1, 32, 256>(p, s);
  else if (nv <= 64) launch_fwd<T, VEC, 2, 32, 256>(p, s);
  else if (nv <= 128) launch_fwd<T, VEC, 4, 32, 256>(p, s);
  else if (nv <= 256) launch_fwd<T, VEC, 2, 128, 256>(p, s);
  else if (nv <= 512) launch_fwd<T, VEC, 2, 256, 256>(p, s);
  else if (nv <= 1024) launch_fwd<T, VEC, 4, 256, 256>(p, s);
  else if (nv <= 2048) launch_fwd<T, VEC, 4, 512, 512>(p, s);
  else if (nv <= 4096) launch_fwd<T, VEC, 4, 1024, 1024>(p, s);
  else return false;
  return true;
}

template <typename T>
int forward(const FwdArgs& p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = p.cols % V == 0 && aligned(p.x, p.xs, V, sizeof(T)) && aligned(p.y, p.ys, V, sizeof(T));
  if (!(vec ? dispatch_fwd<T, V>(p, s) : dispatch_fwd<T, 1>(p, s)))
    layernorm_fwd_loop_kernel<T><<<(unsigned)p.rows, kLoopThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "layernorm forward launch");
}

// Blocks that share the rows of the backward pass: two per SM, never more than there are rows.
int bwd_groups(int64_t rows, int sms) {
  const int64_t g = 2 * (int64_t)sms;
  return (int)(rows < g ? (rows > 0 ? rows : 1) : g);
}

template <typename T, int VEC, int NV, int TPR, int BT>
int launch_bwd(const BwdArgs& p, cudaStream_t s) {
  const int smem = BT / TPR > 1 ? BT * NV * VEC * (int)sizeof(float) : 0;
  layernorm_bwd_kernel<T, VEC, NV, TPR, BT><<<(unsigned)p.groups, BT, smem, s>>>(p);
  return 1;
}

template <typename T, int VEC>
int dispatch_bwd(const BwdArgs& p, cudaStream_t s) {
  const int64_t nv = ((int64_t)p.cols + VEC - 1) / VEC;
  if (nv <= 16) return launch_bwd<T, VEC, 1, 16, 256>(p, s);
  if (nv <= 32) return launch_bwd<T, VEC, 1, 32, 256>(p, s);
  if (nv <= 64) return launch_bwd<T, VEC, 1, 64, 256>(p, s);
  if (nv <= 128) return launch_bwd<T, VEC, 1, 128, 256>(p, s);
  if (nv <= 256) return launch_bwd<T, VEC, 1, 256, 256>(p, s);
  if (nv <= 512) return launch_bwd<T, VEC, 2, 256, 256>(p, s);
  if (nv <= 1024) return launch_bwd<T, VEC, 2, 512, 512>(p, s);
  return 0;
}

template <typename T>
int backward(const BwdArgs& p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = p.cols % V == 0 && aligned(p.x, p.xs, V, sizeof(T)) && aligned(p.dout, p.dos, V, sizeof(T)) &&
                   aligned(p.dx, p.dxs, V, sizeof(T));
  if (!(vec ? dispatch_bwd<T, V>(p, s) : dispatch_bwd<T, 1>(p, s))) {
    layernorm_bwd_loop_kernel<T><<<(unsigned)p.rows, kLoopThreads, 0, s>>>(p);
    if (p.partial)
      layernorm_bwd_columns_kernel<T>
          <<<dim3((unsigned)((p.cols + kColThreads - 1) / kColThreads), (unsigned)p.groups), kColThreads, 0, s>>>(p);
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
  const FwdArgs p{d->x, d->gamma, d->beta, d->y, d->mean, d->rstd, d->rows, d->x_row_stride, d->y_row_stride,
                  (int)d->cols, d->param_dtype == PDB_BF16, (float)d->eps, (float)(1.0 / (double)d->cols)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return d->dtype == PDB_F32 ? forward<float>(p, s) : forward<__nv_bfloat16>(p, s);
}

extern "C" size_t pdb_layernorm_bwd_workspace_size(const pdb_layernorm_bwd_desc* d) {
  if (!d || d->rows < 0 || d->cols <= 0 || d->cols > kMaxCols || !d->dgamma) return 0;
  int dev = 0;
  cudaGetDevice(&dev);
  return (size_t)2 * bwd_groups(d->rows, sm_count(dev)) * d->cols * sizeof(float);
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
  if (d->dgamma && (!d->workspace || d->workspace_bytes < pdb_layernorm_bwd_workspace_size(d)))
    return set_error(PDB_ERR_ARG, "layernorm backward: workspace too small");
  int dev = 0;
  cudaGetDevice(&dev);
  const BwdArgs p{d->dout, d->x, d->mean, d->rstd, d->gamma, d->dx,
                  d->dgamma ? static_cast<float*>(d->workspace) : nullptr, d->rows, d->dout_row_stride,
                  d->x_row_stride, d->dx_row_stride, (int)d->cols, d->param_dtype == PDB_BF16,
                  bwd_groups(d->rows, sm_count(dev)), (float)(1.0 / (double)d->cols)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->rows > 0)
    if (int st = d->dtype == PDB_F32 ? backward<float>(p, s) : backward<__nv_bfloat16>(p, s)) return st;
  if (!d->dgamma) return PDB_OK;
  layernorm_bwd_finish_kernel<<<dim3((unsigned)((d->cols + 31) / 32), 2), 32 * kFinWarps, 0, s>>>(
      p.partial, d->rows > 0 ? p.groups : 0, p.cols, d->dgamma, d->dbeta, p.param_bf16);
  return cuda_status(cudaGetLastError(), "layernorm backward finish launch");
}
