// The cross entropy of a linear head from hidden states x [tokens, width] and the
// head's weight w [vocab, width], without storing the logits, and its gradients.
//
//   logit[n, v] = x[n] . w[v]           lse[n] = log sum_v exp(logit[n, v])
//   loss[n] = lse[n] - logit[n, target[n]]
//   G[n, v] = (exp(logit[n, v] - lse[n]) - [v == target[n]]) dloss[n]
//   dx = G w     dw = G^T x
//
// Forward: one product whose epilogue reduces each row of a tile to a running
// maximum and a sum of exponentials (32 bits), and a small kernel that joins the
// tiles' pairs.  Backward: per piece of the vocabulary, the product again with an
// epilogue that turns logits into G (bf16, the operand type of the two products
// that follow), then dw of the piece, complete in one product, and dx, summed over
// the pieces in f32.
//
// All of it is bound by the tensor cores: 2 (forward) and 6 (backward) x tokens x
// vocab x width operations.  One persistent kernel serves the four products: CTA
// pairs (cta_group::2) on 256 x 256 tiles, operands by TMA into a six-stage ring,
// two f32 accumulators in TMEM so that a tile's epilogue runs under the next
// tile's products.  An operand is read K-major (its rows are the tile's rows) or
// MN-major (its rows are the contracted index): G^T, x and w enter dw and dx that
// way, as they lie in memory.
#include <algorithm>
#include <cfloat>

#include "common.cuh"
#include "tma.h"

namespace pdb {
namespace {

constexpr int TM = 256, TN = 256, TK = 64, STAGES = 6, THREADS = 384;
constexpr int kHalf = 128 * TK * 2;  // one CTA's half of an operand tile, bytes
constexpr int kSmem = STAGES * 2 * kHalf + 256 + 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

enum Epilogue { kStats = 0, kDlogits = 1, kOut = 2 };

struct Args {
  int64_t m, n, k;
  int splits, kb_split;  // shares of the contracted index, and 64-wide blocks in each
  int group;             // m tiles that share a sweep over the n tiles
  int* err;
  // kStats, kDlogits: rows are tokens, columns vocabulary entries from col0 on
  const int64_t* target;
  int64_t col0, ignore, vocab;
  float2* part;   // kStats: (base, sum) per [2 x n tile][m]
  float* tlogit;  // kStats: the target's logit
  const float* lse;
  const float* dloss;
  int64_t dloss_stride;
  const float* unit;   // kDlogits: divides dloss; kOut: multiplies the result (null: 1)
  __nv_bfloat16* out;  // kDlogits: G; kOut: the result, or null when it goes to f32
  int64_t ldo;
  float* acc;  // kOut: f32 [splits][m][n]
  int add;     // kOut: add to acc
};

struct __align__(8) Bars {
  uint64_t full[STAGES], empty[STAGES];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort;
};

// Tile t -> (split, m0, n0): groups of `group` m tiles sweep the n tiles, odd groups backwards, so the tiles
// in flight share operands in L2.
__device__ __forceinline__ void tile_at(const Args& p, int tm, int tn, int64_t t, int& split, int64_t& m0, int64_t& n0) {
  const int64_t per = (int64_t)tm * tn;
  split = (int)(t / per);
  const int64_t r = t - split * per;
  const int64_t gsz = (int64_t)p.group * tn;
  const int grp = (int)(r / gsz);
  const int in = (int)(r - grp * gsz);
  const int rows = min(tm - grp * p.group, p.group);
  const int nt = in / rows;
  m0 = (int64_t)(grp * p.group + in % rows) * TM;
  n0 = (int64_t)((grp & 1) ? tn - 1 - nt : nt) * TN;
}

// One row's 32 logits of a chunk folded into its running maximum and its sum of 2^(logit log2e - base).  The maximum
// is kept as the rounded base itself, so its rounding cancels in lse = (base + log2 sum) ln 2.
__device__ __forceinline__ void fold(const float (&v)[32], float& base, float& s) {
  float c = v[0];
#pragma unroll
  for (int i = 1; i < 31; i += 2) c = max3(c, v[i], v[i + 1]);
  c = fmaxf(c, v[31]);
  const float top = fmaxf(base, c * kLog2e);
  const float b = top == -INFINITY ? 0.f : top;  // nothing but masked columns so far: every term is 0
  s *= ex2(base - b);
  float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 32; ++i) a[i & 3] += ex2(fmaf(v[i], kLog2e, -b));
  s += (a[0] + a[1]) + (a[2] + a[3]);
  base = top;
}

template <bool A_MN, bool B_MN, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    linear_ce_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                          const __grid_constant__ Args p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * kHalf;
  Bars* bar = reinterpret_cast<Bars*>(sB + STAGES * kHalf);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int nk = (int)((p.k + TK - 1) / TK);
  const int tm = (int)((p.m + TM - 1) / TM), tn = (int)((p.n + TN - 1) / TN);
  const int64_t num_tiles = (int64_t)tm * tn * p.splits;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->acc_full[i], 1);
      mbar_init(&bar->acc_empty[i], 16);  // one arrival per epilogue warp of the pair
    }
    bar->abort = 0;
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc_pair(&bar->tmem_base, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;
  volatile int* abort = &bar->abort;

  if (warp == 0 && lane == 0) {
    uint32_t g = 0;
    bool ok = true;
    for (int64_t t = pair; ok && t < num_tiles; t += npairs) {
      int split;
      int64_t m0, n0;
      tile_at(p, tm, tn, t, split, m0, n0);
      const int kb0 = split * p.kb_split, kb1 = min(nk, kb0 + p.kb_split);
      const int ma = (int)m0 + (int)rank * 128, nb = (int)n0 + (int)rank * 128;
      for (int kb = kb0; kb < kb1; ++kb, ++g) {
        const int st = g % STAGES;
        if (!(ok = mbar_wait_cluster(&bar->empty[st], ((g / STAGES) & 1) ^ 1, abort, p.err))) break;
        if (rank == 0) mbar_expect_tx(&bar->full[st], 4 * kHalf);
        const uint32_t full0 = mapa_shared(smem_u32(&bar->full[st]), 0);
        uint8_t *a = sA + st * kHalf, *b = sB + st * kHalf;
        if constexpr (A_MN) {  // two boxes of 64 tile rows x 64 contracted rows
          tma_load_4d_pair(a, &tm_a, full0, ma, kb * TK, 0, 0);
          tma_load_4d_pair(a + kHalf / 2, &tm_a, full0, ma + 64, kb * TK, 0, 0);
        } else {
          tma_load_4d_pair(a, &tm_a, full0, kb * TK, ma, 0, 0);
        }
        if constexpr (B_MN) {
          tma_load_4d_pair(b, &tm_b, full0, nb, kb * TK, 0, 0);
          tma_load_4d_pair(b + kHalf / 2, &tm_b, full0, nb + 64, kb * TK, 0, 0);
        } else {
          tma_load_4d_pair(b, &tm_b, full0, kb * TK, nb, 0, 0);
        }
      }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    constexpr uint32_t idesc = idesc_bf16(TM, TN, A_MN, B_MN);
    // K-major: a step of 16 is 32 bytes along the swizzled row; MN-major: 16 rows of 128 bytes, the
    // second 64 columns in the next box
    constexpr uint32_t a_step = A_MN ? 2048 : 32, a_lbo = A_MN ? kHalf / 2 : 16;
    constexpr uint32_t b_step = B_MN ? 2048 : 32, b_lbo = B_MN ? kHalf / 2 : 16;
    uint32_t g = 0, tt = 0;
    bool ok = true;
    for (int64_t t = pair; ok && t < num_tiles; t += npairs, ++tt) {
      const int split = (int)(t / ((int64_t)tm * tn));
      const int kb0 = split * p.kb_split, kb1 = min(nk, kb0 + p.kb_split);
      const int buf = tt & 1;
      if (!(ok = mbar_wait_cluster(&bar->acc_empty[buf], ((tt >> 1) & 1) ^ 1, abort, p.err))) break;
      tc_fence_after();
      const uint32_t acc = tmem + buf * TN;
      for (int kb = kb0; kb < kb1; ++kb, ++g) {
        const int st = g % STAGES;
        if (!(ok = mbar_wait_cluster(&bar->full[st], (g / STAGES) & 1, abort, p.err))) break;
        tc_fence_after();
        const uint32_t a0 = smem_u32(sA + st * kHalf), b0 = smem_u32(sB + st * kHalf);
#pragma unroll
        for (int kk = 0; kk < TK / 16; ++kk)
          mma_ss_pair(acc, sdesc_sw128(a0 + kk * a_step, a_lbo, 1024), sdesc_sw128(b0 + kk * b_step, b_lbo, 1024), idesc,
                      (kb > kb0 || kk > 0) ? 1u : 0u);
        const uint32_t e = smem_u32(&bar->empty[st]);
        tc_commit_pair(e);
        tc_commit_pair(mapa_shared(e, 1));
      }
      if (ok) {
        const uint32_t f = smem_u32(&bar->acc_full[buf]);
        tc_commit_pair(f);
        tc_commit_pair(mapa_shared(f, 1));
      }
    }
  } else if (warp >= 4) {
    const int q4 = warp & 3, half = (warp - 4) >> 2;  // TMEM lane quarter, column half
    const int row = (int)rank * 128 + q4 * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    uint32_t tt = 0;
    for (int64_t t = pair; t < num_tiles; t += npairs, ++tt) {
      int split;
      int64_t m0, n0;
      tile_at(p, tm, tn, t, split, m0, n0);
      const int buf = tt & 1;
      const int64_t gm = m0 + row;
      const bool live = gm < p.m;
      int64_t tgt = -1;
      float nlse = 0.f, up = 0.f;
      bool skip = false;
      if constexpr (EPI != kOut) {
        if (live) {
          tgt = p.target[gm];
          skip = tgt == p.ignore;
          if constexpr (EPI == kDlogits) {
            nlse = -p.lse[gm] * kLog2e;
            up = p.dloss[gm * p.dloss_stride] / *p.unit;
            if (!skip && (tgt < 0 || tgt >= p.vocab)) up = NAN;  // no such entry: the gradient says so
          }
          tgt -= p.col0;
        }
      }
      if (!mbar_wait_cluster(&bar->acc_full[buf], (tt >> 1) & 1, abort, p.err)) break;
      tc_fence_after();
      float mx = -INFINITY, sum = 0.f;
      const float unit = EPI == kOut && p.unit ? *p.unit : 1.f;
#pragma unroll 1
      for (int ch = half * (TN / 64); ch < (half + 1) * (TN / 64); ++ch) {
        uint32_t r[32];
        __syncwarp();  // rows past the end left the last chunk early
        tmem_ld32(tmem + lane_off + buf * TN + ch * 32, r);
        tmem_wait_ld();
        const int64_t c0 = n0 + ch * 32;
        if (!live || c0 >= p.n) continue;
        const int nv = (int)min((int64_t)32, p.n - c0);
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        const int hit = (int)max((int64_t)-1, min((int64_t)32, tgt - c0));
        if constexpr (EPI == kStats) {
          if (hit >= 0 && hit < nv) {
            float x = v[0];
#pragma unroll
            for (int i = 1; i < 32; ++i) x = i == hit ? v[i] : x;
            p.tlogit[gm] = x;
          }
          if (nv < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = i < nv ? v[i] : -INFINITY;
          }
          fold(v, mx, sum);
        } else {
          __nv_bfloat16* C = nullptr;
          if constexpr (EPI == kDlogits) {
            C = p.out + gm * p.ldo + c0;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float g = (ex2(fmaf(v[i], kLog2e, nlse)) - (i == hit ? 1.f : 0.f)) * up;
              v[i] = skip ? 0.f : g;
            }
          } else {
            if (p.acc) {
              float* dst = p.acc + ((int64_t)split * p.m + gm) * p.n + c0;
              if ((p.n & 3) == 0 && nv == 32) {
                float4* d4 = reinterpret_cast<float4*>(dst);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  float4 o = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                  if (p.add) {
                    const float4 q = d4[i];
                    o.x += q.x, o.y += q.y, o.z += q.z, o.w += q.w;
                  }
                  d4[i] = o;
                }
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (i < nv) dst[i] = p.add ? dst[i] + v[i] : v[i];
              }
              continue;
            }
            C = p.out + gm * p.ldo + c0;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= unit;
          }
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
          if (nv == 32 && (p.ldo & 7) == 0) {
            uint4* dst = reinterpret_cast<uint4*>(C);
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[i] = make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < nv) C[i] = __ushort_as_bfloat16((unsigned short)(pk[i >> 1] >> (16 * (i & 1))));
          }
        }
      }
      if constexpr (EPI == kStats)
        if (live) p.part[((n0 / TN) * 2 + half) * p.m + gm] = make_float2(mx, sum);
      warp_arrive_cluster_after_tc(mapa_shared(smem_u32(&bar->acc_empty[buf]), 0));
    }
  }
  tc_fence_before();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Joins a row's (base, sum) pairs: one warp per row.
constexpr int kFinishWarps = 4;

__global__ void __launch_bounds__(32 * kFinishWarps)
    linear_ce_finish_kernel(const float2* part, int parts, const float* tlogit, const int64_t* target, int64_t tokens,
                            int64_t vocab, int64_t ignore, float* loss, float* lse) {
  const int64_t row = (int64_t)blockIdx.x * kFinishWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= tokens) return;
  float m = -INFINITY, s = 0.f;
  for (int i = lane; i < parts; i += 32) {
    const float2 q = part[(int64_t)i * tokens + row];
    const float mn = fmaxf(m, q.x);
    if (mn != -INFINITY) s = s * exp2f(m - mn) + q.y * exp2f(q.x - mn);
    m = mn;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float mo = __shfl_xor_sync(0xffffffffu, m, o), so = __shfl_xor_sync(0xffffffffu, s, o);
    const float mn = fmaxf(m, mo);
    if (mn != -INFINITY) s = s * exp2f(m - mn) + so * exp2f(mo - mn);
    m = mn;
  }
  if (lane == 0) {
    const float l = (m + log2f(s)) * kLn2;
    const int64_t t = target[row];
    if (lse) lse[row] = l;
    if (loss) loss[row] = t == ignore ? 0.f : (t < 0 || t >= vocab) ? NAN : l - tlogit[row];
  }
}

// The unit that dloss is measured in: its largest finite magnitude over the tokens that count (1 if that is 0).  G
// is rounded to bf16 in this unit.  In dloss's own units the entries of all targets, -(1 - p) dloss with p near 0,
// would under a mean be one and the same number, whose rounding (up to 2^-9) would not average out but scale the
// whole gradient; in this unit it is 1, which is exact.
__global__ void __launch_bounds__(1024)
    linear_ce_unit_kernel(const float* dloss, int64_t stride, const int64_t* target, int64_t ignore, int64_t tokens, float* unit) {
  __shared__ float red[32];
  float m = 0.f;
  for (int64_t i = threadIdx.x; i < tokens; i += 1024) {
    const float a = fabsf(dloss[i * stride]);
    if (target[i] != ignore && a <= FLT_MAX) m = fmaxf(m, a);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x < 32) {
    m = red[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (threadIdx.x == 0) *unit = m > 0.f ? m : 1.f;
  }
}

// The f32 shares of a product, added in order and rounded.
__global__ void __launch_bounds__(256)
    linear_ce_join_kernel(const float* acc, int splits, int64_t m, int64_t n, const float* unit, __nv_bfloat16* out,
                          int64_t ldo) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;  // n is a multiple of 8
  if (i >= m * n) return;
  float4 s = *reinterpret_cast<const float4*>(acc + i);
  for (int k = 1; k < splits; ++k) {
    const float4 q = *reinterpret_cast<const float4*>(acc + (int64_t)k * m * n + i);
    s.x += q.x, s.y += q.y, s.z += q.z, s.w += q.w;
  }
  const float u = *unit;
  uint2 o = make_uint2(pack_bf16(s.x * u, s.y * u), pack_bf16(s.z * u, s.w * u));
  *reinterpret_cast<uint2*>(out + (i / n) * ldo + i % n) = o;
}

// ------------------------------------------------------------------- host
int map2d(CUtensorMap* map, const void* base, int64_t inner, int64_t rows, int64_t ld, int box_inner, int box_rows) {
  const uint64_t dims[4] = {(uint64_t)inner, (uint64_t)rows, 1, 1};
  const uint64_t str[3] = {(uint64_t)ld * 2, (uint64_t)ld * 2, (uint64_t)ld * 2};
  const uint32_t box[4] = {(uint32_t)box_inner, (uint32_t)box_rows, 1, 1};
  return encode_tma_4d(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

struct Matrix {  // rows x cols as they lie in memory, ld elements apart
  const void* p;
  int64_t rows, cols, ld;
};

int pair_count() {
  int dev = 0;
  cudaGetDevice(&dev);
  return std::max(1, sm_count(dev) / 2);
}

// One product: a.m x b.n over k.  K-major operands have k columns, MN-major ones k rows.
template <bool A_MN, bool B_MN, int EPI>
int gemm(const Matrix& a, const Matrix& b, Args p, cudaStream_t s) {
  CUtensorMap ta, tb;
  if (int st = map2d(&ta, a.p, a.cols, a.rows, a.ld, 64, A_MN ? 64 : 128)) return st;
  if (int st = map2d(&tb, b.p, b.cols, b.rows, b.ld, 64, B_MN ? 64 : 128)) return st;
  p.err = device_error_flag();
  auto kernel = linear_ce_gemm_kernel<A_MN, B_MN, EPI>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem))
    return cuda_status(e, "linear cross entropy: smem attribute");
  const int64_t tiles = ((p.m + TM - 1) / TM) * ((p.n + TN - 1) / TN) * p.splits;
  const int64_t pairs = std::min<int64_t>(tiles, pair_count());
  kernel<<<(unsigned)(2 * pairs), THREADS, kSmem, s>>>(ta, tb, p);
  return cuda_status(cudaGetLastError(), "linear cross entropy launch");
}

constexpr int64_t kAlign = 256;
int64_t up256(int64_t n) { return (n + kAlign - 1) / kAlign * kAlign; }
int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Sizes up to here keep every product below within 2^62.
constexpr int64_t kMaxTokens = 1 << 24, kMaxVocab = 1 << 24, kMaxWidth = 1 << 16;

int check(int64_t tokens, int64_t vocab, int64_t width, int64_t x_stride, int64_t w_stride, int32_t dtype) {
  if (dtype != PDB_BF16)
    return set_error(PDB_ERR_UNSUPPORTED, "linear cross entropy: built for bf16 operands only (dtype %d)", dtype);
  if (tokens < 0 || vocab <= 0 || width <= 0)
    return set_error(PDB_ERR_SHAPE, "linear cross entropy: vocab and width must be positive, tokens not negative");
  if (tokens > kMaxTokens || vocab > kMaxVocab || width > kMaxWidth)
    return set_error(PDB_ERR_SHAPE, "linear cross entropy: at most 2^24 tokens and entries, width 2^16");
  if (width % 8 != 0) return set_error(PDB_ERR_ALIGN, "linear cross entropy: width must be a multiple of 8");
  if (x_stride < width || w_stride < width || x_stride % 8 != 0 || w_stride % 8 != 0)
    return set_error(PDB_ERR_ALIGN, "linear cross entropy: row strides must be multiples of 8 and at least width");
  return PDB_OK;
}

struct FwdPlan {
  int parts;
  int64_t part, tlogit, bytes;  // byte offsets
};
FwdPlan plan_fwd(int64_t tokens, int64_t vocab) {
  FwdPlan f{};
  f.parts = (int)(2 * div_up(vocab, TN));
  f.tlogit = up256((int64_t)f.parts * tokens * 8);
  f.bytes = f.tlogit + up256(tokens * 4);
  return f;
}

// Shares of the contracted index for a product that has fewer tiles than there are CTA pairs: each
// share at least 8 blocks of 64.
void split_k(Args& p, int pairs, int64_t k) {
  const int64_t tiles = div_up(p.m, TM) * div_up(p.n, TN), nk = div_up(k, TK);
  int64_t s = std::max<int64_t>(1, std::min(pairs / tiles, nk / 8));
  p.kb_split = (int)div_up(nk, s);
  p.splits = (int)div_up(nk, p.kb_split);
}

struct BwdPlan {
  int64_t piece, pieces;  // vocabulary entries per piece
  int dx_splits, dw_splits;
  int64_t g, unit, dx_acc, dw_acc, bytes;
};
// G of one piece: at most this many bytes
constexpr int64_t kPieceBytes = int64_t(512) << 20;

BwdPlan plan_bwd(int64_t tokens, int64_t vocab, int64_t width, int pairs) {
  BwdPlan b{};
  const int64_t most = std::max<int64_t>(TN, kPieceBytes / (2 * std::max<int64_t>(tokens, 1)) / TN * TN);
  b.pieces = div_up(vocab, most);
  b.piece = std::min(div_up(div_up(vocab, b.pieces), TN) * TN, div_up(vocab, 8) * 8);
  b.pieces = div_up(vocab, b.piece);
  Args a{};
  a.m = tokens, a.n = width;
  split_k(a, pairs, std::min(b.piece, vocab));
  b.dx_splits = a.splits;
  a.m = std::min(b.piece, vocab);
  split_k(a, pairs, tokens);
  b.dw_splits = a.splits;
  int64_t at = up256(tokens * b.piece * 2);
  b.unit = at;
  at += kAlign;
  b.dx_acc = at;
  if (b.dx_splits > 1 || b.pieces > 1) at += up256(b.dx_splits * tokens * width * 4);
  b.dw_acc = at;
  if (b.dw_splits > 1) at += up256(b.dw_splits * std::min(b.piece, vocab) * width * 4);
  b.bytes = at;
  return b;
}

void join(const float* acc, int splits, int64_t m, int64_t n, const float* unit, void* out, int64_t ldo, cudaStream_t s) {
  linear_ce_join_kernel<<<(unsigned)div_up(m * n, 1024), 256, 0, s>>>(acc, splits, m, n, unit,
                                                                       static_cast<__nv_bfloat16*>(out), ldo);
}

bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace pdb

using namespace pdb;

extern "C" size_t pdb_linear_ce_fwd_workspace_size(const pdb_linear_ce_fwd_desc* d) {
  if (!d || check(d->tokens, d->vocab, d->width, d->x_stride, d->w_stride, d->dtype) != PDB_OK || d->tokens == 0) return 0;
  return (size_t)plan_fwd(d->tokens, d->vocab).bytes;
}

extern "C" int pdb_linear_ce_fwd(const pdb_linear_ce_fwd_desc* d, void* stream) {
  if (!d) return set_error(PDB_ERR_ARG, "null descriptor");
  if (int st = check(d->tokens, d->vocab, d->width, d->x_stride, d->w_stride, d->dtype)) return st;
  if (d->tokens == 0) return PDB_OK;
  if (!d->x || !d->w || !d->target || (!d->loss && !d->lse))
    return set_error(PDB_ERR_ARG, "linear cross entropy: null x / w / target, or neither loss nor lse");
  const FwdPlan f = plan_fwd(d->tokens, d->vocab);
  if (!d->workspace || d->workspace_bytes < (size_t)f.bytes || !a16(d->workspace))
    return set_error(PDB_ERR_ARG, "linear cross entropy: workspace too small or not 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(d->workspace);
  Args p{};
  p.m = d->tokens;
  p.n = d->vocab;
  p.k = d->width;
  p.splits = 1;
  p.kb_split = (int)div_up(d->width, TK);
  p.group = 8;
  p.target = d->target;
  p.ignore = d->ignore_index;
  p.vocab = d->vocab;
  p.part = reinterpret_cast<float2*>(ws + f.part);
  p.tlogit = reinterpret_cast<float*>(ws + f.tlogit);
  const Matrix x{d->x, d->tokens, d->width, d->x_stride}, w{d->w, d->vocab, d->width, d->w_stride};
  if (int st = gemm<false, false, kStats>(x, w, p, s)) return st;
  linear_ce_finish_kernel<<<(unsigned)div_up(d->tokens, kFinishWarps), 32 * kFinishWarps, 0, s>>>(
      p.part, f.parts, p.tlogit, d->target, d->tokens, d->vocab, d->ignore_index, d->loss, d->lse);
  return cuda_status(cudaGetLastError(), "linear cross entropy finish launch");
}

extern "C" size_t pdb_linear_ce_bwd_workspace_size(const pdb_linear_ce_bwd_desc* d) {
  if (!d || check(d->tokens, d->vocab, d->width, d->x_stride, d->w_stride, d->dtype) != PDB_OK || d->tokens == 0) return 0;
  return (size_t)plan_bwd(d->tokens, d->vocab, d->width, pair_count()).bytes;
}

extern "C" int pdb_linear_ce_bwd(const pdb_linear_ce_bwd_desc* d, void* stream) {
  if (!d) return set_error(PDB_ERR_ARG, "null descriptor");
  if (int st = check(d->tokens, d->vocab, d->width, d->x_stride, d->w_stride, d->dtype)) return st;
  if (d->dx && (d->dx_stride < d->width || d->dx_stride % 8 != 0 || !a16(d->dx)))
    return set_error(PDB_ERR_ALIGN, "linear cross entropy: dx must be 16-byte aligned with a row stride that is a multiple of 8");
  if (d->dw && (d->dw_stride < d->width || d->dw_stride % 8 != 0 || !a16(d->dw)))
    return set_error(PDB_ERR_ALIGN, "linear cross entropy: dw must be 16-byte aligned with a row stride that is a multiple of 8");
  if (!d->dx && !d->dw) return set_error(PDB_ERR_ARG, "linear cross entropy: neither dx nor dw");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->tokens == 0) {  // nothing adds to dw
    if (!d->dw) return PDB_OK;
    return cuda_status(cudaMemset2DAsync(d->dw, d->dw_stride * 2, 0, d->width * 2, d->vocab, s), "linear cross entropy: zero dw");
  }
  if (!d->x || !d->w || !d->target || !d->lse || !d->dloss)
    return set_error(PDB_ERR_ARG, "linear cross entropy: null x / w / target / lse / dloss");
  const BwdPlan b = plan_bwd(d->tokens, d->vocab, d->width, pair_count());
  if (!d->workspace || d->workspace_bytes < (size_t)b.bytes || !a16(d->workspace))
    return set_error(PDB_ERR_ARG, "linear cross entropy: workspace too small or not 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(d->workspace);
  float* dx_acc = reinterpret_cast<float*>(ws + b.dx_acc);
  float* dw_acc = reinterpret_cast<float*>(ws + b.dw_acc);
  float* unit = reinterpret_cast<float*>(ws + b.unit);
  linear_ce_unit_kernel<<<1, 1024, 0, s>>>(d->dloss, d->dloss_stride, d->target, d->ignore_index, d->tokens, unit);
  if (int st = cuda_status(cudaGetLastError(), "linear cross entropy unit launch")) return st;
  const Matrix x{d->x, d->tokens, d->width, d->x_stride};
  for (int64_t i = 0; i < b.pieces; ++i) {
    const int64_t v0 = i * b.piece, nv = std::min(b.piece, d->vocab - v0);
    const Matrix w{static_cast<const __nv_bfloat16*>(d->w) + v0 * d->w_stride, nv, d->width, d->w_stride};
    const Matrix g{ws, d->tokens, nv, b.piece};
    Args p{};
    p.group = 8;
    p.m = d->tokens;
    p.n = nv;
    p.k = d->width;
    p.splits = 1;
    p.kb_split = (int)div_up(d->width, TK);
    p.target = d->target;
    p.col0 = v0;
    p.ignore = d->ignore_index;
    p.vocab = d->vocab;
    p.lse = d->lse;
    p.dloss = d->dloss;
    p.dloss_stride = d->dloss_stride;
    p.unit = unit;
    p.out = reinterpret_cast<__nv_bfloat16*>(ws);
    p.ldo = b.piece;
    if (int st = gemm<false, false, kDlogits>(x, w, p, s)) return st;
    if (d->dw) {
      Args q{};
      q.group = 8;
      q.m = nv;
      q.n = d->width;
      q.k = d->tokens;
      q.kb_split = (int)div_up(div_up(q.k, TK), b.dw_splits);
      q.splits = (int)div_up(div_up(q.k, TK), q.kb_split);
      q.out = static_cast<__nv_bfloat16*>(d->dw) + v0 * d->dw_stride;
      q.ldo = d->dw_stride;
      q.unit = unit;
      if (q.splits > 1) q.acc = dw_acc;
      if (int st = gemm<true, true, kOut>(g, x, q, s)) return st;
      if (q.acc) join(q.acc, q.splits, q.m, q.n, unit, q.out, q.ldo, s);
    }
    if (d->dx) {
      Args q{};
      q.group = 8;
      q.m = d->tokens;
      q.n = d->width;
      q.k = nv;
      // every piece takes the same number of shares, so that each share has its own sum
      const int64_t nk = div_up(nv, TK);
      q.kb_split = (int)div_up(nk, b.dx_splits);
      q.splits = (int)div_up(nk, q.kb_split);
      q.out = static_cast<__nv_bfloat16*>(d->dx);
      q.ldo = d->dx_stride;
      q.unit = unit;
      if (b.dx_splits > 1 || b.pieces > 1) q.acc = dx_acc;
      q.add = i > 0;
      if (int st = gemm<false, true, kOut>(g, w, q, s)) return st;
    }
  }
  if (d->dx && (b.dx_splits > 1 || b.pieces > 1)) join(dx_acc, b.dx_splits, d->tokens, d->width, unit, d->dx, d->dx_stride, s);
  return cuda_status(cudaGetLastError(), "linear cross entropy join launch");
}
