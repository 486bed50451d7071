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
// tiles' pairs.  Backward: the tokens that are ignored are left out first (their rows
// of x are not even read by the products, whatever they hold), by a kernel that packs
// the others' rows and counts them; the products take the count from memory.  Then,
// per piece of the vocabulary, the product again with an epilogue that turns logits
// into G (bf16, the operand type of the two products that follow), dw of the piece,
// complete in one product, and dx, summed over the pieces in f32.
//
// All of it is bound by the tensor cores: 2 (forward) and 6 (backward) x tokens x
// vocab x width operations.  One persistent kernel serves the four products: tiles of
// 256 rows on CTA pairs (cta_group::2), or of 128 rows on single CTAs where the rows
// make an odd number of 128-row blocks up to seven, by up to 256 columns; operands by
// TMA into a ring, two f32 accumulators in TMEM so that a tile's epilogue runs under
// the next tile's products.
// An operand is read K-major (its rows are the tile's rows) or MN-major (its rows are
// the contracted index): G^T, x and w enter dw and dx that way, as they lie in memory.
// Sixteen warps run the epilogue, 64 columns of 32 rows each, and hand results to TMA
// stores through shared memory (rows of dx whose tokens were packed go to their places
// by 16-byte stores).  On a B200, 4096 tokens x 65536 x 2048: the loss in 676 us cool
// (1.63 PFLOP/s), 820 warm under the power limit (1.34); 8192 x 128000 x 4096 gradients
// with a tenth ignored in 16.4 ms cool, 18.4 warm (1.41 and 1.26 PFLOP/s of the tokens
// that count).
//
// f32 operands take the same steps on IEEE multiply-adds (the f32 column refuses
// reduced operand types): linear_ce_f32_kernel, G in f32.
#include <algorithm>
#include <cfloat>
#include <utility>

#include "common.cuh"
#include "tma.h"

namespace pdb {
namespace {

constexpr int TK = 64, kEpiWarps = 16, THREADS = 128 + 32 * kEpiWarps;
constexpr int kBox = 64 * 64 * 2;      // an MN-major box: 64 tile rows x 64 contracted rows
constexpr int kTileA = 128 * TK * 2;   // a CTA's rows of A per stage
constexpr int kStore = 4096;           // an epilogue warp's staging: 32 rows x 64 bf16 or 32 f32, 128-byte swizzle
                                       // (kStats: 128 rows' (base, sum) of three of the four groups of columns)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

enum Epilogue { kStats = 0, kDlogits = 1, kOut = 2, kSum = 3 };  // kOut: bf16, kSum: f32

// CG: CTAs per tile.  Each holds 128 rows of A; B's rows are split between the CTAs of a pair.
template <int CG, int EPI>
struct Layout {
  static constexpr int kTileB = 256 / CG * TK * 2;
  static constexpr int kStage = kTileA + kTileB;
  static constexpr int kStaging = EPI == kStats ? 3 * 128 * 8 + 1024 : kEpiWarps * kStore;
  static constexpr int kStages = (227 * 1024 - 1024 - 256 - kStaging) / kStage;
  static constexpr int kSmem = kStages * kStage + kStaging + 256 + 1024;
};

struct Args {
  int64_t m, n, k;
  int tile_n;            // columns per tile, a multiple of 64 (of 32 for kStats), at most 256
  int splits, kb_split;  // shares of the contracted index, and 64-wide blocks in each
  int group;             // m tiles that share a sweep over the n tiles
  int* err;
  // The tokens that count, found on the device: state[0] of them; state[1]: their rows of x are packed, under tm_x.
  const int* state;      // null: all of them, unpacked
  int dyn;               // 1: m, 2: k is their number
  const int* token_of;   // kOut: the row of the result that each packed row goes to
  __nv_bfloat16* out;    // ... and the result
  int64_t ldo;
  // kStats, kDlogits: rows are (packed) tokens, columns vocabulary entries from col0 on
  const int64_t* target;
  int64_t col0, vocab;
  float2* part;        // kStats: (base, sum) per [n tile][m]
  float* tlogit;       // kStats: the target's logit
  const float* lse;    // kDlogits
  const float* dloss;
  const float* unit;   // kDlogits: the unit that G is measured in; kOut: multiplies the result
  int add;             // kSum: add to what is there
};

struct __align__(8) Bars {
  uint64_t full[8], empty[8];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t left[4], taken[4];  // kStats, per 32 rows
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(Bars) <= 256, "the barriers' share of shared memory");

// Tile t -> (split, m0, n0): groups of `group` m tiles sweep the n tiles, odd groups backwards, so the tiles
// in flight share operands in L2.  In 32 bits: every epilogue warp does this for every tile.
template <int TM>
__device__ __forceinline__ void tile_at(const Args& p, uint32_t tm, uint32_t tn, uint32_t t, int& split, int& m0, int& n0) {
  const uint32_t per = tm * tn;
  split = (int)(t / per);
  const uint32_t r = t - split * per;
  const uint32_t gsz = p.group * tn;
  const uint32_t grp = r / gsz, in = r - grp * gsz;
  const uint32_t rows = min(tm - grp * p.group, (uint32_t)p.group);
  const uint32_t nt = in / rows;
  m0 = (int)(grp * p.group + in - nt * rows) * TM;
  n0 = (int)((grp & 1) ? tn - 1 - nt : nt) * p.tile_n;
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
  const uint64_t l2 = f2_pack(kLog2e, kLog2e), nb = f2_pack(-b, -b);
  uint64_t a0 = f2_pack(0.f, 0.f), a1 = a0;
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    float x, y, z, w;
    f2_unpack(f2_fma(f2_pack(v[i], v[i + 1]), l2, nb), x, y);
    f2_unpack(f2_fma(f2_pack(v[i + 2], v[i + 3]), l2, nb), z, w);
    a0 = f2_add(a0, f2_pack(ex2(x), ex2(y)));
    a1 = f2_add(a1, f2_pack(ex2(z), ex2(w)));
  }
  float lo, hi;
  f2_unpack(f2_add(a0, a1), lo, hi);
  s += lo + hi;
  base = top;
}

// Two (base, sum) pairs into one.
__device__ __forceinline__ void join_sums(float2& a, float2 b) {
  const float m = fmaxf(a.x, b.x), z = m == -INFINITY ? 0.f : m;
  a = make_float2(m, a.y * exp2f(a.x - z) + b.y * exp2f(b.x - z));
}

// The products issued so far arrive on this barrier (of both CTAs of a pair) when they are done.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
  else
    tc_commit(bar);
}

// A warp's accumulator columns are read (tmem_wait_ld has returned): one arrival at rank 0's barrier.  Relaxed, since
// nothing but tensor memory is handed over: a release at cluster scope waits for all of the warp's memory traffic.
__device__ __forceinline__ void warp_arrive_rank0(uint64_t* bar) {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  if ((threadIdx.x & 31) == 0)
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(mapa_shared(smem_u32(bar), 0)) : "memory");
}

template <int CG, bool A_MN, bool B_MN, int EPI>
__global__ void __launch_bounds__(THREADS, 1)
    linear_ce_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                          const __grid_constant__ CUtensorMap tm_c, const __grid_constant__ CUtensorMap tm_x,
                          const __grid_constant__ Args p) {
  using L = Layout<CG, EPI>;
  constexpr int TM = 128 * CG, STAGES = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * kTileA;
  uint8_t* sC = sB + STAGES * L::kTileB;
  Bars* bar = reinterpret_cast<Bars*>(sC + L::kStaging);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const int unit_id = blockIdx.x / CG, units = gridDim.x / CG;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
    if constexpr (EPI != kStats) prefetch_tensormap(&tm_c);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->acc_full[i], 1);
      mbar_init(&bar->acc_empty[i], CG * kEpiWarps);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bar->left[i], 3);
      mbar_init(&bar->taken[i], 1);
    }
    bar->abort = 0;
    fence_barrier_init();
  }
  if (warp == 2) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(&bar->tmem_base, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&bar->tmem_base, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  grid_dep_wait();  // the launch before may still be writing what this one reads
  const uint32_t tmem = bar->tmem_base;
  volatile int* abort = &bar->abort;
  int64_t m = p.m, k = p.k;
  bool packed = false, scatter = false;
  if (EPI != kStats && p.state) {
    const int count = p.state[0];
    packed = p.state[1] != 0;
    scatter = p.dyn == 1 && count < m;
    (p.dyn == 1 ? m : k) = count;
  }
  const int nk = (int)((k + TK - 1) / TK), kb_split = p.dyn == 2 ? (nk + p.splits - 1) / p.splits : p.kb_split;
  const int tm = (int)((m + TM - 1) / TM), tn = (int)((p.n + p.tile_n - 1) / p.tile_n);
  const int num_tiles = tm * tn * p.splits;  // the host saw to it that they are fewer than 2^31

  if (warp == 0 && lane == 0) {
    const int b_rows = p.tile_n / CG;  // of B per CTA
    const CUtensorMap* map_a = EPI == kDlogits && packed ? &tm_x : &tm_a;
    const CUtensorMap* map_b = A_MN && packed ? &tm_x : &tm_b;
    const uint32_t bytes = CG * (kTileA + b_rows * TK * 2);
    uint32_t g = 0;
    bool ok = true;
    for (int t = unit_id; ok && t < num_tiles; t += units) {
      int split, m0, n0;
      tile_at<TM>(p, tm, tn, t, split, m0, n0);
      const int kb0 = split * kb_split, kb1 = min(nk, kb0 + kb_split);
      const int ma = m0 + (int)rank * 128, nb = n0 + (int)rank * b_rows;
      for (int kb = kb0; kb < kb1; ++kb, ++g) {
        const int st = g % STAGES;
        if (!(ok = mbar_wait(&bar->empty[st], ((g / STAGES) & 1) ^ 1, abort, p.err))) break;
        if (rank == 0) mbar_expect_tx(&bar->full[st], bytes);
        const uint32_t full0 = CG == 2 ? mapa_shared(smem_u32(&bar->full[st]), 0) : 0;
        auto load = [&](uint8_t* dst, const CUtensorMap* map, int c0, int c1) {
          if constexpr (CG == 2) tma_load_4d_pair(dst, map, full0, c0, c1, 0, 0);
          else tma_load_4d(dst, map, &bar->full[st], c0, c1, 0, 0);
        };
        uint8_t *a = sA + st * kTileA, *b = sB + st * L::kTileB;
        if constexpr (A_MN) {
          load(a, map_a, ma, kb * TK);
          load(a + kBox, map_a, ma + 64, kb * TK);
        } else {
          load(a, map_a, kb * TK, ma);
        }
        if constexpr (B_MN) {
          for (int r = 0; r < b_rows; r += 64) load(b + r / 64 * kBox, map_b, nb + r, kb * TK);
        } else {
          load(b, map_b, kb * TK, nb);
        }
      }
    }
    // given up: this thread's copies in flight arrive first (a pair's are counted at rank 0, and its CTAs leave together)
    if (!ok && rank == 0) {
      int never = 0;
      for (uint32_t i = g > STAGES ? g - STAGES : 0; i < g; ++i)
        mbar_wait(&bar->full[i % STAGES], (i / STAGES) & 1, &never, nullptr, 10000000ull);
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    const uint32_t idesc = idesc_bf16(TM, 0, A_MN, B_MN) | ((uint32_t)(p.tile_n >> 3) << 17);
    // K-major: a step of 16 is 32 bytes along the swizzled row; MN-major: 16 rows of 128 bytes, the
    // next 64 columns in the next box
    constexpr uint32_t a_step = A_MN ? 2048 : 32, a_lbo = A_MN ? kBox : 16;
    constexpr uint32_t b_step = B_MN ? 2048 : 32, b_lbo = B_MN ? kBox : 16;
    // The loop is kept short: its scheduler also serves epilogue warps, and a block's four products are over in 512 cycles.
    // A descriptor's start address counts 16 bytes, so a stage and a step are additions to its low word.
    const uint64_t da0 = sdesc_sw128(smem_u32(sA), a_lbo, 1024), db0 = sdesc_sw128(smem_u32(sB), b_lbo, 1024);
    uint32_t st = 0, parity = 0, tt = 0;
    bool ok = true;
    for (int t = unit_id; ok && t < num_tiles; t += units, ++tt) {
      const int split = (int)((uint32_t)t / (uint32_t)(tm * tn));
      const int kb0 = split * kb_split, kb1 = min(nk, kb0 + kb_split);
      const int buf = tt & 1;
      if (!(ok = mbar_wait(&bar->acc_empty[buf], ((tt >> 1) & 1) ^ 1, abort, p.err))) break;
      tc_fence_after();
      const uint32_t acc = tmem + buf * 256;
      uint32_t more = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = mbar_wait(&bar->full[st], parity, abort, p.err))) break;
        tc_fence_after();
        const uint64_t da = da0 + st * (kTileA >> 4), db = db0 + st * (L::kTileB >> 4);
#pragma unroll
        for (int kk = 0; kk < TK / 16; ++kk) {
          if constexpr (CG == 2) mma_ss_pair(acc, da + (kk * a_step >> 4), db + (kk * b_step >> 4), idesc, more | kk);
          else mma_ss(acc, da + (kk * a_step >> 4), db + (kk * b_step >> 4), idesc, more | kk);
        }
        more = 1;
        commit<CG>(&bar->empty[st]);
        if (++st == STAGES) st = 0, parity ^= 1;
      }
      if (ok) commit<CG>(&bar->acc_full[buf]);
    }
  } else if (warp >= 4) {
    const int e = warp - 4, q4 = warp & 3, cg = e >> 2;  // TMEM lane quarter, group of 64 columns
    const int row0 = (int)rank * 128 + q4 * 32;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    const uint32_t stage = smem_u32(sC + e * kStore), srow = stage + lane * 128;
    float unit = 1.f;
    if constexpr (EPI == kDlogits || EPI == kOut) unit = *p.unit;
    // the next tile's place and its rows' targets, lse and dloss, found while the tile before is worked on
    int next_split = 0, next_m0 = 0, next_n0 = 0;
    int64_t next_target = -1;
    float next_lse = 0.f, next_dloss = 0.f;
    auto look = [&](int t) {
      if (t >= num_tiles) return;
      tile_at<TM>(p, tm, tn, t, next_split, next_m0, next_n0);
      if constexpr (EPI == kStats || EPI == kDlogits) {
        const int row = next_m0 + row0 + lane;
        if (row >= m) return;
        next_target = p.target[row];
        if constexpr (EPI == kDlogits) next_lse = p.lse[row], next_dloss = p.dloss[row];
      }
    };
    look(unit_id);
    uint32_t tt = 0;
    for (int t = unit_id; t < num_tiles; t += units, ++tt) {
      const int split = next_split, m0 = next_m0, n0 = next_n0;
      const int buf = tt & 1;
      const int64_t gm = m0 + row0 + lane;  // rows and columns are below 2^25
      const bool live = gm < m;
      const bool none = split * kb_split >= nk;  // a share of the contracted index without any of it
      // the target's column in this tile, if it is there
      const int64_t away = next_target - p.col0 - n0;
      const int tgt = live && away >= 0 && away < 256 ? (int)away : -256;
      const float nlse = -next_lse * kLog2e;
      float up = next_dloss / unit;
      if (next_target < 0 || next_target >= p.vocab) up = NAN;  // no such entry: the gradient says so
      look(t + units);
      if (!mbar_wait(&bar->acc_full[buf], (tt >> 1) & 1, abort, p.err)) break;
      tc_fence_after();
      float base = -INFINITY, sum = 0.f;
#pragma unroll 1
      for (int ch = 0; ch < 2; ++ch) {
        const int c = cg * 64 + ch * 32;  // the tile's column
        const int c0 = n0 + c;
        if (c >= p.tile_n || c0 >= p.n) break;  // the whole warp
        uint32_t r[32];
        __syncwarp();
        tmem_ld32(tmem + lane_off + buf * 256 + c, r);
        tmem_wait_ld();
        if ((EPI == kOut || EPI == kSum) && none) {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0u;
        }
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        const int hit = tgt - c;  // 0 .. 31: in this chunk
        if constexpr (EPI == kStats) {
          const int nv = (int)min((int64_t)32, p.n - c0);
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
          fold(v, base, sum);
        } else if constexpr (EPI == kSum) {
          // 32 columns fill the staging: 128 bytes a row
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) sts128(srow + ((i ^ (lane & 7)) << 4), r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && m0 + row0 < m) {
            if (p.add) tma_reduce_add_4d(&tm_c, stage, c0, m0 + row0, split, 0);
            else tma_store_4d(&tm_c, stage, c0, m0 + row0, split, 0);
            bulk_commit();
          }
        } else {
          if constexpr (EPI == kDlogits) {
            const uint64_t l2 = f2_pack(kLog2e, kLog2e), nl = f2_pack(nlse, nlse);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float x, y;
              f2_unpack(f2_fma(f2_pack(v[i], v[i + 1]), l2, nl), x, y);
              v[i] = ex2(x);
              v[i + 1] = ex2(y);
            }
            if (hit >= 0 && hit < 32) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = i == hit ? v[i] - 1.f : v[i];
            }
          }
          const float scale = EPI == kDlogits ? up : unit;
          const uint64_t s2 = f2_pack(scale, scale);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x, y;
            f2_unpack(f2_mul(f2_pack(v[2 * i], v[2 * i + 1]), s2), x, y);
            pk[i] = pack_bf16(x, y);
          }
          if (EPI == kDlogits && m0 + row0 + 32 > m) {  // rows behind the last token, whatever their accumulators hold
#pragma unroll
            for (int i = 0; i < 16; ++i) pk[i] = live ? pk[i] : 0u;
          }
          if (ch == 0) {
            if (lane == 0) bulk_wait_read_all();
            __syncwarp();
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sts128(srow + (((ch * 4 + i) ^ (lane & 7)) << 4), pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
        }
      }
      if constexpr (EPI == kOut || EPI == kDlogits) {
        // the box is cut at the last row and column by its tensor map
        // (rows of G behind the last token are 0 up to the end of a block of 64, which dw sums over)
        const int64_t rows = EPI == kDlogits ? min(p.m, (m + TK - 1) / TK * TK) : m;
        if (cg * 64 < p.tile_n && n0 + cg * 64 < p.n && m0 + row0 < rows) {
          fence_proxy_async_smem();
          __syncwarp();
          if (EPI == kOut && !A_MN && scatter) {  // eight lanes per row, four rows at a time, each to its token's row
            const int64_t col = n0 + cg * 64 + (lane & 7) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i * 4 + (lane >> 3);
              const int64_t row = m0 + row0 + r;
              uint4 q;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                           : "r"(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4))
                           : "memory");
              if (row < m && col < p.n) *reinterpret_cast<uint4*>(p.out + p.token_of[row] * p.ldo + col) = q;
            }
          } else if (lane == 0) {
            tma_store_4d(&tm_c, stage, n0 + cg * 64, m0 + row0, 0, 0);
            bulk_commit();
          }
        }
      }
      if constexpr (CG == 2) warp_arrive_rank0(&bar->acc_empty[buf]);
      else warp_arrive_after_tc(&bar->acc_empty[buf]);
      if constexpr (EPI == kStats) {
        // the four warps with these rows join their columns: three leave theirs in shared memory for the first
        float2* mine = reinterpret_cast<float2*>(sC) + q4 * 32 + lane;
        if (cg > 0) {
          if (tt > 0 && !mbar_wait(&bar->taken[q4], (tt - 1) & 1, abort, p.err)) break;
          mine[(cg - 1) * 128] = make_float2(base, sum);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->left[q4]);
        } else {
          if (!mbar_wait(&bar->left[q4], tt & 1, abort, p.err)) break;
          float2 j = make_float2(base, sum);
#pragma unroll
          for (int i = 0; i < 3; ++i) join_sums(j, mine[i * 128]);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->taken[q4]);
          if (live) p.part[(int64_t)(n0 / p.tile_n) * m + gm] = j;
        }
      }
    }
    if (EPI != kStats && lane == 0) bulk_wait_all();
  }
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync_all();
  else __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// Joins the rows' (base, sum) pairs: a block takes 32 rows (a lane each) and its 32 warps a share of the pairs each.
constexpr int kFinishWarps = 32;

__global__ void __launch_bounds__(32 * kFinishWarps)
    linear_ce_finish_kernel(const float2* part, int parts, const float* tlogit, const int64_t* target, int64_t tokens,
                            int64_t vocab, int64_t ignore, float* loss, float* lse) {
  __shared__ float2 red[kFinishWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * 32 + lane;
  grid_dep_wait();
  float2 s = make_float2(-INFINITY, 0.f);
  if (row < tokens) {
    constexpr int FLIGHT = 8;  // loads before the first is joined
    for (int i = warp; i < parts; i += FLIGHT * kFinishWarps) {
      float2 q[FLIGHT];
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) {
        const int k = i + u * kFinishWarps;
        q[u] = k < parts ? part[(int64_t)k * tokens + row] : make_float2(-INFINITY, 0.f);
      }
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) join_sums(s, q[u]);
    }
  }
  red[warp][lane] = s;
  __syncthreads();
  // turned: a warp joins one row's 32 shares
  s = red[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float2 q = make_float2(__shfl_xor_sync(0xffffffffu, s.x, o), __shfl_xor_sync(0xffffffffu, s.y, o));
    join_sums(s, q);
  }
  const int64_t r = (int64_t)blockIdx.x * 32 + warp;
  if (lane == 0 && r < tokens) {
    const float l = (s.x + log2f(s.y)) * kLn2;
    const int64_t t = target[r];
    if (lse) lse[r] = l;
    if (loss) loss[r] = t == ignore ? 0.f : (t < 0 || t >= vocab) ? NAN : l - tlogit[r];
  }
}

// The f32 shares of a product, added in a fixed order, scaled and rounded; packed rows go to their tokens' rows.
// GROUPS threads share an element's shares (one after another, 135 shares of a small product took 38 us).
constexpr int kJoinThreads = 256;

template <int GROUPS, typename T>
__global__ void __launch_bounds__(kJoinThreads)
    linear_ce_join_kernel(const float* acc, int splits, int64_t m, int64_t n, const float* unit, const int* state,
                          const int* token_of, T* out, int64_t ldo) {
  constexpr int EACH = kJoinThreads / GROUPS, FLIGHT = 8;
  __shared__ float4 red[GROUPS][EACH];
  const int group = threadIdx.x / EACH, l = threadIdx.x % EACH;
  const int64_t i = ((int64_t)blockIdx.x * EACH + l) * 4;  // n is a multiple of 4
  grid_dep_wait();
  const bool live = i < (state ? *state : m) * n;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    for (int k = group; k < splits; k += FLIGHT * GROUPS) {
      float4 q[FLIGHT];
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) {
        const int at = k + u * GROUPS;
        q[u] = at < splits ? *reinterpret_cast<const float4*>(acc + (int64_t)at * m * n + i) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) s.x += q[u].x, s.y += q[u].y, s.z += q[u].z, s.w += q[u].w;
    }
  }
  if constexpr (GROUPS > 1) {
    red[group][l] = s;
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) {
      const float4 q = red[g][l];
      s.x += q.x, s.y += q.y, s.z += q.z, s.w += q.w;
    }
  }
  if (!live) return;
  const int64_t row = i / n;
  T* at = out + (token_of ? token_of[row] : row) * ldo + i % n;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(at) = s;
  } else {
    const float u = *unit;
    *reinterpret_cast<uint2*>(at) = make_uint2(pack_bf16(s.x * u, s.y * u), pack_bf16(s.z * u, s.w * u));
  }
}

// Packs the tokens that count, in their order: their rows of x (when a token is ignored, or `pack`: rows that do not
// start on 128-byte lines cost the products a quarter more reads), targets, lse and dloss; and writes their number, the
// rows of dx that stay 0, and the unit of dloss.
//
// The unit is dloss's largest finite magnitude over those tokens (1 if that is 0).  G is rounded to bf16 in this unit.
// In dloss's own units the entries of all targets, -(1 - p) dloss with p near 0, would under a mean be one and the same
// number, whose rounding (up to 2^-9) would not average out but scale the whole gradient; in this unit it is 1, which
// is exact.
//
// A block packs `rows` tokens; for its place it counts the tokens before them itself, so one launch is enough.
template <typename T>
struct Pack {
  const T* x;
  const int64_t* target;
  const float* lse;
  const float* dloss;
  int64_t tokens, width, ldx, dloss_stride, ignore;
  int rows, pack;
  T* xp;  // [tokens][ldp]
  int64_t ldp;
  int64_t* targetp;
  float* lsep;
  float* dlossp;
  int* token_of;
  int* state;
  float* unit;
  T* dx;  // nullable
  int64_t lddx;
};

constexpr int kPackThreads = 512, kPackWarps = kPackThreads / 32;

template <typename T>
__global__ void __launch_bounds__(kPackThreads) linear_ce_pack_kernel(const Pack<T> p) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ int before_s[kPackWarps], total_s[kPackWarps], place[kPackThreads];
  __shared__ float max_s[kPackWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t first = (int64_t)blockIdx.x * p.rows, last = min(p.tokens, first + p.rows);
  grid_dep_wait();
  int before = 0, total = 0;
  float top = 0.f;
  constexpr int FLIGHT = 16;  // loads before the first is looked at: the count is all latency
  for (int i = tid; i < (int)p.tokens; i += FLIGHT * kPackThreads) {
    int64_t t[FLIGHT];
    float a[FLIGHT];
#pragma unroll
    for (int u = 0; u < FLIGHT; ++u) {
      const int n = i + u * kPackThreads;
      t[u] = n < (int)p.tokens ? p.target[n] : p.ignore;
      a[u] = n < (int)p.tokens && blockIdx.x == 0 ? fabsf(p.dloss[n * p.dloss_stride]) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < FLIGHT; ++u) {
      const bool counts = t[u] != p.ignore;
      before += counts && i + u * kPackThreads < first;
      total += counts;
      if (counts && a[u] <= FLT_MAX) top = fmaxf(top, a[u]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (lane == 0) before_s[warp] = before, total_s[warp] = total, max_s[warp] = top;
  __syncthreads();
  before = total = 0;
  for (int i = 0; i < kPackWarps; ++i) before += before_s[i], total += total_s[i], top = fmaxf(top, max_s[i]);
  const bool pack = p.pack || total < p.tokens;
  if (blockIdx.x == 0 && tid == 0) {
    p.state[0] = total;
    p.state[1] = pack;
    *p.unit = top > 0.f ? top : 1.f;
  }
  const int64_t vecs = p.width / VEC;
  for (int64_t c = first; c < last; c += kPackThreads) {
    const int64_t n = c + tid;
    const bool counts = n < last && p.target[n] != p.ignore;
    const uint32_t votes = __ballot_sync(0xffffffffu, counts);
    __syncthreads();
    if (lane == 0) before_s[warp] = __popc(votes);
    __syncthreads();
    int at = before + __popc(votes & ((1u << lane) - 1u)), all = 0;
    for (int i = 0; i < kPackWarps; ++i) {
      at += i < warp ? before_s[i] : 0;
      all += before_s[i];
    }
    before += all;
    place[tid] = counts ? at : -1;
    if (counts) {
      p.targetp[at] = p.target[n];
      p.lsep[at] = p.lse[n];
      p.dlossp[at] = p.dloss[n * p.dloss_stride];
      p.token_of[at] = (int)n;
    }
    __syncthreads();
    if (!pack) continue;
    const int64_t here = min((int64_t)kPackThreads, last - c);
    for (int64_t e = tid; e < here * vecs; e += kPackThreads) {
      const int r = (int)(e / vecs);
      const int64_t col = (e - r * vecs) * VEC;
      if (place[r] >= 0)
        *reinterpret_cast<uint4*>(p.xp + place[r] * p.ldp + col) = *reinterpret_cast<const uint4*>(p.x + (c + r) * p.ldx + col);
      else if (p.dx)
        *reinterpret_cast<uint4*>(p.dx + (c + r) * p.lddx + col) = make_uint4(0, 0, 0, 0);
    }
  }
  // the rest of the last block of 64 rows that dw sums over: G is 0 there, and x must not be infinite
  if (pack && blockIdx.x == gridDim.x - 1) {
    const int64_t rest = min(p.tokens, (int64_t)(total + TK - 1) / TK * TK) - total;
    for (int64_t e = tid; e < rest * vecs; e += kPackThreads)
      *reinterpret_cast<uint4*>(p.xp + (total + e / vecs) * p.ldp + e % vecs * VEC) = make_uint4(0, 0, 0, 0);
  }
}

// ---------------------------------------------------------------- f32 path
// The same four products on IEEE multiply-adds (two per instruction): 128 x 128 tiles, 16 deep, 8 x 8 per thread (two
// groups of four rows and of four columns, so that shared memory is read 16 bytes wide without conflicts), the next
// block's loads in flight; two blocks per SM, and a long contraction under few tiles in shares that join() adds up.
// The FMA pipes bound it: 4096 tokens of 1024 x 32000 entries take 6.0 ms (44.5 TFLOP/s; 8.7 ms with one multiply-add per
// instruction and one block per SM) and their gradients 18.3 ms (44.0; 26.1); 64 tokens of 512 x 8000 entries' gradients
// take 0.13 ms (0.98 before).
constexpr int FT = 128, FK = 16, FTHREADS = 256;

struct F32Args {
  const float *a, *b;
  int64_t m, n, k, lda, ldb;
  const float* xp;  // packed rows of x: a of G, b of dw, when state[1]
  int64_t ldp;
  const int* state;
  int dyn;  // as in Args
  const int* token_of;
  const int64_t* target;
  int64_t col0, vocab;
  float2* part;  // [n tile][m]
  float* tlogit;
  const float *lse, *dloss;
  float* out;
  int64_t ldo;
  int add;
  int splits;  // > 1: out is [splits][m][n], a share of the contracted index each
};

template <bool A_MN, bool B_MN, int EPI>
__global__ void __launch_bounds__(FTHREADS, 2) linear_ce_f32_kernel(const F32Args p) {
  __shared__ __align__(16) float As[2][FK][FT + 4], Bs[2][FK][FT + 4];
  grid_dep_wait();
  int64_t m = p.m, k = p.k, lda = p.lda, ldb = p.ldb;
  const float *A = p.a, *B = p.b;
  if (EPI != kStats && p.state) {
    (p.dyn == 1 ? m : k) = p.state[0];
    if (p.state[1]) {
      if (EPI == kDlogits) A = p.xp, lda = p.ldp;
      if (A_MN) B = p.xp, ldb = p.ldp;
    }
  }
  const uint32_t tm = (uint32_t)((p.m + FT - 1) / FT);  // the grid's, whatever the number of tokens is
  const int64_t m0 = (int64_t)(blockIdx.x % tm) * FT, n0 = (int64_t)(blockIdx.x / tm) * FT;
  if (m0 >= m) return;
  // this block's share of the contracted index: [k1, k)
  const int64_t share = ((k + FK - 1) / FK + p.splits - 1) / p.splits * FK, k1 = blockIdx.y * share;
  k = min(k, k1 + share);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  // four elements along the operand's rows in memory; what lies outside the product is 0
  auto load = [&](const float* x, int64_t ld, bool mn, int64_t first, int64_t rows, int64_t k0, int i) {
    const int e = tid + i * FTHREADS;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mn) {
      const int64_t kk = k0 + (e >> 5), r = first + (e & 31) * 4;
      if (kk < k && r < rows) v = *reinterpret_cast<const float4*>(x + kk * ld + r);
    } else {
      const int64_t r = first + (e >> 2), kk = k0 + (e & 3) * 4;
      if (r < rows && kk < k) {
        v = *reinterpret_cast<const float4*>(x + r * ld + kk);
        if (kk + 1 >= k) v.y = 0.f;
        if (kk + 2 >= k) v.z = 0.f;
        if (kk + 3 >= k) v.w = 0.f;
      }
    }
    return v;
  };
  auto store = [&](float (&s)[FK][FT + 4], bool mn, const float4& v, int i) {
    const int e = tid + i * FTHREADS;
    if (mn) {
      *reinterpret_cast<float4*>(&s[e >> 5][(e & 31) * 4]) = v;
    } else {
      const int r = e >> 2, kk = (e & 3) * 4;
      s[kk][r] = v.x, s[kk + 1][r] = v.y, s[kk + 2][r] = v.z, s[kk + 3][r] = v.w;
    }
  };
  uint64_t acc2[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc2[i][j] = f2_pack(0.f, 0.f);
  float4 av[2], bv[2];
  auto fetch = [&](int64_t k0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) av[i] = load(A, lda, A_MN, m0, m, k0, i), bv[i] = load(B, ldb, B_MN, n0, p.n, k0, i);
  };
  fetch(k1);
  int buf = 0;
  for (int64_t k0 = k1; k0 < k; k0 += FK, buf ^= 1) {
#pragma unroll
    for (int i = 0; i < 2; ++i) store(As[buf], A_MN, av[i], i), store(Bs[buf], B_MN, bv[i], i);
    __syncthreads();  // the other buffer was read before the barrier of the block before
    if (k0 + FK < k) fetch(k0 + FK);
#pragma unroll
    for (int kk = 0; kk < FK; ++kk) {
      float a[8];
      uint64_t b2[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 x = *reinterpret_cast<const float4*>(&As[buf][kk][h * 64 + ty * 4]);
        const float4 y = *reinterpret_cast<const float4*>(&Bs[buf][kk][h * 64 + tx * 4]);
        a[4 * h] = x.x, a[4 * h + 1] = x.y, a[4 * h + 2] = x.z, a[4 * h + 3] = x.w;
        b2[2 * h] = f2_pack(y.x, y.y), b2[2 * h + 1] = f2_pack(y.z, y.w);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint64_t a2 = f2_pack(a[i], a[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc2[i][j] = f2_fma(a2, b2[j], acc2[i][j]);
      }
    }
  }
  float acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) f2_unpack(acc2[i][j], acc[i][2 * j], acc[i][2 * j + 1]);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = m0 + (i >> 2) * 64 + ty * 4 + (i & 3);
    const bool live = row < m;
    const int64_t tgt = EPI != kOut && live ? p.target[row] : -1;
    if constexpr (EPI == kStats) {
      float2 s = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t col = n0 + (j >> 2) * 64 + tx * 4 + (j & 3);
        if (col >= p.n) acc[i][j] = -INFINITY;
        else if (col == tgt) p.tlogit[row] = acc[i][j];
        s.x = fmaxf(s.x, acc[i][j] * kLog2e);
      }
      const float base = s.x == -INFINITY ? 0.f : s.x;
#pragma unroll
      for (int j = 0; j < 8; ++j) s.y += exp2f(fmaf(acc[i][j], kLog2e, -base));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1)
        join_sums(s, make_float2(__shfl_xor_sync(0xffffffffu, s.x, o), __shfl_xor_sync(0xffffffffu, s.y, o)));
      if (tx == 0 && live) p.part[n0 / FT * m + row] = s;
    } else if (live) {
      const float lse = EPI == kDlogits ? p.lse[row] : 0.f;
      // an index that the vocabulary does not have: the gradient says so
      const float up = EPI != kDlogits ? 1.f : tgt < 0 || tgt >= p.vocab ? NAN : p.dloss[row];
      float* to = p.out + blockIdx.y * p.m * p.ldo + (EPI == kOut && p.token_of ? p.token_of[row] : row) * p.ldo;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t col = n0 + h * 64 + tx * 4;
        if (col >= p.n) continue;  // rows of the result reach the next multiple of four columns
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = acc[i][4 * h + j];
          if constexpr (EPI == kDlogits) v[j] = (expf(v[j] - lse) - (col + j + p.col0 == tgt ? 1.f : 0.f)) * up;
        }
        float4* at = reinterpret_cast<float4*>(to + col);
        if (EPI == kOut && p.add) {
          const float4 q = *at;
          v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
        }
        *at = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
  }
}

// ------------------------------------------------------------------- host
struct Matrix {  // rows x cols as they lie in memory, ld elements apart
  const void* p;
  int64_t rows, cols, ld;
};

int map2d(CUtensorMap* map, const Matrix& x, int box_inner, int box_rows) {
  const uint64_t dims[4] = {(uint64_t)x.cols, (uint64_t)x.rows, 1, 1};
  const uint64_t str[3] = {(uint64_t)x.ld * 2, (uint64_t)x.ld * 2, (uint64_t)x.ld * 2};
  const uint32_t box[4] = {(uint32_t)box_inner, (uint32_t)box_rows, 1, 1};
  return encode_tma_4d(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x.p, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int sms() {
  int dev = 0;
  cudaGetDevice(&dev);
  return std::max(2, sm_count(dev));
}

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Launched behind the grid before it: set-up overlaps that grid's tail, and every kernel waits before it reads.
template <typename... Params, typename... Given>
int launch(void (*kernel)(Params...), dim3 grid, int threads, int smem, int cluster, cudaStream_t s, Given&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, std::forward<Given>(args)...), "linear cross entropy launch");
}

// A pair's tile has 256 rows: where they end in an odd block of 128, and few come before it, single CTAs waste less than
// they lose by reading B alone (300 x 32000 x 2048: 49 us against 60 on pairs; 640: 73 against 83; 256: 56 against 53).
int cta_group(int64_t m) {
  const int64_t blocks = div_up(m, 128);
  return blocks % 2 == 1 && blocks <= 7 ? 1 : 2;
}

// The tile's width: of the multiples of `step`, the one whose waves of tiles load least, since operand rows into shared
// memory (the tile's rows and its columns) are what a step costs: at 1024 x 50176 x 1024, 17 waves of 160 columns took
// 105 us where 11 waves of 256 take 84.
int tile_width(int64_t m, int64_t n, int splits, int step, int units) {
  const int rows = 128 * cta_group(m);
  const int64_t tm = div_up(m, rows);
  int best = 256;
  int64_t least = 0;
  for (int w = 256; w >= 64; w -= step) {
    const int64_t work = div_up(tm * div_up(n, w) * splits, units) * (rows + w);
    if (w == 256 || work < least) best = w, least = work;
  }
  return best;
}

// One product: a.m x b.n over k.  K-major operands have k columns, MN-major ones k rows.  xp: the packed rows of x
// (A of G, B of dw), where the product has a choice.
template <int CG, bool A_MN, bool B_MN, int EPI>
int gemm_on(const Matrix& a, const Matrix& b, const CUtensorMap& tc, const Matrix& xp, Args p, cudaStream_t s) {
  using L = Layout<CG, EPI>;
  p.tile_n = tile_width(p.m, p.n, p.splits, EPI == kStats && !B_MN ? 32 : 64 * CG, sms() / CG);
  CUtensorMap ta, tb, tx{};
  if (xp.p)
    if (int st = map2d(&tx, xp, 64, A_MN ? 64 : 128)) return st;
  if (int st = map2d(&ta, a, 64, A_MN ? 64 : 128)) return st;
  if (int st = map2d(&tb, b, 64, B_MN ? 64 : p.tile_n / CG)) return st;
  p.err = device_error_flag();
  p.group = 8;
  auto kernel = linear_ce_gemm_kernel<CG, A_MN, B_MN, EPI>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem))
    return cuda_status(e, "linear cross entropy: smem attribute");
  const int64_t tiles = div_up(p.m, 128 * CG) * div_up(p.n, p.tile_n) * p.splits;
  if (tiles > 0x3fffffffLL) return set_error(PDB_ERR_SHAPE, "linear cross entropy: too many tiles");
  return launch(kernel, CG * std::min<int64_t>(tiles, sms() / CG), THREADS, L::kSmem, CG, s, ta, tb, tc, tx, p);
}

template <bool A_MN, bool B_MN, int EPI>
int gemm(const Matrix& a, const Matrix& b, const CUtensorMap& tc, const Matrix& xp, const Args& p, cudaStream_t s) {
  return cta_group(p.m) == 1 ? gemm_on<1, A_MN, B_MN, EPI>(a, b, tc, xp, p, s)
                             : gemm_on<2, A_MN, B_MN, EPI>(a, b, tc, xp, p, s);
}

// ... whose result goes to bf16, or to f32 shares [splits][m][n] when acc is given.
template <bool A_MN, bool B_MN>
int gemm_out(const Matrix& a, const Matrix& b, const Matrix& out, float* acc, const Matrix& xp, Args p, cudaStream_t s) {
  CUtensorMap tc;
  if (!acc) {
    if (int st = map2d(&tc, out, 64, 32)) return st;
    p.out = static_cast<__nv_bfloat16*>(const_cast<void*>(out.p));
    p.ldo = out.ld;
    return gemm<A_MN, B_MN, kOut>(a, b, tc, xp, p, s);
  }
  const uint64_t dims[4] = {(uint64_t)p.n, (uint64_t)p.m, (uint64_t)p.splits, 1};
  const uint64_t str[3] = {(uint64_t)p.n * 4, (uint64_t)(p.m * p.n) * 4, (uint64_t)(p.m * p.n) * 4};
  const uint32_t box[4] = {32, 32, 1, 1};
  if (int st = encode_tma_4d(&tc, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, acc, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) return st;
  return gemm<A_MN, B_MN, kSum>(a, b, tc, xp, p, s);
}

constexpr int64_t kAlign = 256;
int64_t up256(int64_t n) { return (n + kAlign - 1) / kAlign * kAlign; }
// Sizes up to here keep every product below within 2^62.
constexpr int64_t kMaxTokens = 1 << 24, kMaxVocab = 1 << 24, kMaxWidth = 1 << 16;

int check(int64_t tokens, int64_t vocab, int64_t width, int64_t x_stride, int64_t w_stride, int32_t dtype) {
  if (dtype != PDB_BF16 && dtype != PDB_F32)
    return set_error(PDB_ERR_UNSUPPORTED, "linear cross entropy: unknown dtype %d", dtype);
  const int vec = dtype == PDB_BF16 ? 8 : 4;
  if (tokens < 0 || vocab <= 0 || width <= 0)
    return set_error(PDB_ERR_SHAPE, "linear cross entropy: vocab and width must be positive, tokens not negative");
  if (tokens > kMaxTokens || vocab > kMaxVocab || width > kMaxWidth)
    return set_error(PDB_ERR_SHAPE, "linear cross entropy: at most 2^24 tokens and entries, width 2^16");
  if (width % vec != 0 || x_stride < width || w_stride < width || x_stride % vec != 0 || w_stride % vec != 0)
    return set_error(PDB_ERR_ALIGN,
                     "linear cross entropy: width and row strides must be multiples of 16 bytes, strides at least width");
  return PDB_OK;
}

struct FwdPlan {
  int parts;
  int64_t tlogit, bytes;  // byte offset of the targets' logits
};
FwdPlan plan_fwd(int64_t tokens, int64_t vocab, int32_t dtype) {
  FwdPlan f{};
  const int w = dtype == PDB_F32 ? FT : tile_width(tokens, vocab, 1, 32, sms() / cta_group(tokens));
  f.parts = (int)div_up(vocab, w);
  f.tlogit = up256((int64_t)f.parts * tokens * 8);
  f.bytes = f.tlogit + up256(tokens * 4);
  return f;
}

// Shares of the contracted index for a product that has fewer tiles than there are CTAs or pairs of them: each
// share at least 8 blocks of 64.
void split_k(Args& p, int64_t k) {
  const int cg = cta_group(p.m);
  const int64_t tiles = div_up(p.m, 128 * cg) * div_up(p.n, 256), nk = div_up(k, TK);
  int64_t s = std::max<int64_t>(1, std::min(sms() / cg / tiles, nk / 8));
  p.kb_split = (int)div_up(nk, s);
  p.splits = (int)div_up(nk, p.kb_split);
}

// ... for the f32 products, whose tiles are one block each: shares of at least 16 blocks of 16.
int f32_splits(int64_t m, int64_t n, int64_t k) {
  const int64_t tiles = div_up(m, FT) * div_up(n, FT);
  return (int)std::max<int64_t>(1, std::min<int64_t>({2 * sms() / tiles, div_up(k, FK) / 16, 1024}));
}

struct BwdPlan {
  int64_t piece, pieces;  // vocabulary entries per piece
  int dx_splits, dw_splits;
  int64_t ldp;            // row distance of the packed x
  int64_t state, unit, xp, target, lse, dloss, token_of, dx_acc, dw_acc, bytes;
};
// G of one piece: at most this many bytes
constexpr int64_t kPieceBytes = int64_t(512) << 20;

BwdPlan plan_bwd(int64_t tokens, int64_t vocab, int64_t width, int32_t dtype) {
  BwdPlan b{};
  const int64_t size = dtype == PDB_F32 ? 4 : 2;
  const int64_t most = std::max<int64_t>(256, kPieceBytes / (size * std::max<int64_t>(tokens, 1)) / 256 * 256);
  b.pieces = div_up(vocab, most);
  // rows of G on 128-byte lines: with 50024 columns, 1021 x 50021 x 1000 took 94 us for dx
  b.piece = std::min(div_up(div_up(vocab, b.pieces), 256) * 256, div_up(vocab, 64) * 64);
  b.pieces = div_up(vocab, b.piece);
  Args a{};
  a.m = tokens, a.n = width;
  split_k(a, std::min(b.piece, vocab));
  b.dx_splits = a.splits;
  a.m = std::min(b.piece, vocab);
  split_k(a, tokens);
  b.dw_splits = a.splits;
  if (dtype == PDB_F32) {
    b.dx_splits = f32_splits(tokens, width, std::min(b.piece, vocab));
    b.dw_splits = f32_splits(std::min(b.piece, vocab), width, tokens);
  }
  int64_t at = up256(tokens * b.piece * size);
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up256(bytes);
    return here;
  };
  b.ldp = div_up(width, 64) * 64;
  b.state = take(2 * sizeof(int));
  b.unit = take(sizeof(float));
  b.xp = take(tokens * b.ldp * size);
  b.target = take(tokens * 8);
  b.lse = take(tokens * 4);
  b.dloss = take(tokens * 4);
  b.token_of = take(tokens * 4);
  b.dx_acc = at;
  if (b.dx_splits > 1 || (size == 2 && b.pieces > 1)) at += up256(b.dx_splits * tokens * width * 4);
  b.dw_acc = at;
  if (b.dw_splits > 1) at += up256(b.dw_splits * std::min(b.piece, vocab) * width * 4);
  b.bytes = at;
  return b;
}

template <typename T>
int join(const float* acc, int splits, int64_t m, int64_t n, const float* unit, const int* state, const int* token_of, T* out,
         int64_t ldo, cudaStream_t s) {
  auto on = [&](auto kernel, int groups) {
    return launch(kernel, div_up(m * n, 4 * kJoinThreads / groups), kJoinThreads, 0, 1, s, acc, splits, m, n, unit, state,
                  token_of, out, ldo);
  };
  return splits > 8 ? on(linear_ce_join_kernel<16, T>, 16) : on(linear_ce_join_kernel<1, T>, 1);
}

template <typename T>
int pack(const pdb_linear_ce_bwd_desc& d, const BwdPlan& b, uint8_t* ws, cudaStream_t s) {
  Pack<T> k{};
  k.x = static_cast<const T*>(d.x);
  k.target = d.target;
  k.lse = d.lse;
  k.dloss = d.dloss;
  k.tokens = d.tokens;
  k.width = d.width;
  k.ldx = d.x_stride;
  k.dloss_stride = d.dloss_stride;
  k.ignore = d.ignore_index;
  k.rows = (int)div_up(d.tokens, 2 * sms());
  k.pack = sizeof(T) == 2 && d.width % 64 != 0;
  k.xp = reinterpret_cast<T*>(ws + b.xp);
  k.ldp = b.ldp;
  k.targetp = reinterpret_cast<int64_t*>(ws + b.target);
  k.lsep = reinterpret_cast<float*>(ws + b.lse);
  k.dlossp = reinterpret_cast<float*>(ws + b.dloss);
  k.token_of = reinterpret_cast<int*>(ws + b.token_of);
  k.state = reinterpret_cast<int*>(ws + b.state);
  k.unit = reinterpret_cast<float*>(ws + b.unit);
  k.dx = static_cast<T*>(d.dx);
  k.lddx = d.dx_stride;
  return launch(linear_ce_pack_kernel<T>, div_up(d.tokens, k.rows), kPackThreads, 0, 1, s, k);
}

F32Args f32_product(const Matrix& a, const Matrix& b, int64_t m, int64_t n, int64_t k) {
  F32Args p{};
  p.a = static_cast<const float*>(a.p);
  p.b = static_cast<const float*>(b.p);
  p.m = m;
  p.n = n;
  p.k = k;
  p.lda = a.ld;
  p.ldb = b.ld;
  p.splits = 1;
  return p;
}

template <bool A_MN, bool B_MN, int EPI>
int f32_gemm(const F32Args& p, cudaStream_t s) {
  const int64_t tiles = div_up(p.m, FT) * div_up(p.n, FT);
  if (tiles > 0x7fffffffLL) return set_error(PDB_ERR_SHAPE, "linear cross entropy: too many tiles");
  return launch(linear_ce_f32_kernel<A_MN, B_MN, EPI>, dim3((unsigned)tiles, p.splits), FTHREADS, 0, 1, s, p);
}

bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace pdb

using namespace pdb;

extern "C" size_t pdb_linear_ce_fwd_workspace_size(const pdb_linear_ce_fwd_desc* d) {
  if (!d || check(d->tokens, d->vocab, d->width, d->x_stride, d->w_stride, d->dtype) != PDB_OK || d->tokens == 0) return 0;
  return (size_t)plan_fwd(d->tokens, d->vocab, d->dtype).bytes;
}

extern "C" int pdb_linear_ce_fwd(const pdb_linear_ce_fwd_desc* d, void* stream) {
  if (!d) return set_error(PDB_ERR_ARG, "null descriptor");
  if (int st = check(d->tokens, d->vocab, d->width, d->x_stride, d->w_stride, d->dtype)) return st;
  if (d->tokens == 0) return PDB_OK;
  if (!d->x || !d->w || !d->target || (!d->loss && !d->lse))
    return set_error(PDB_ERR_ARG, "linear cross entropy: null x / w / target, or neither loss nor lse");
  if (!a16(d->x) || !a16(d->w))
    return set_error(PDB_ERR_ALIGN, "linear cross entropy: x and w must be 16-byte aligned");
  const FwdPlan f = plan_fwd(d->tokens, d->vocab, d->dtype);
  if (!d->workspace || d->workspace_bytes < (size_t)f.bytes || !a16(d->workspace))
    return set_error(PDB_ERR_ARG, "linear cross entropy: workspace too small or not 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(d->workspace);
  float2* part = reinterpret_cast<float2*>(ws);
  float* tlogit = reinterpret_cast<float*>(ws + f.tlogit);
  const Matrix x{d->x, d->tokens, d->width, d->x_stride}, w{d->w, d->vocab, d->width, d->w_stride};
  if (d->dtype == PDB_F32) {
    F32Args p = f32_product(x, w, d->tokens, d->vocab, d->width);
    p.target = d->target;
    p.vocab = d->vocab;
    p.part = part;
    p.tlogit = tlogit;
    if (int st = f32_gemm<false, false, kStats>(p, s)) return st;
  } else {
    Args p{};
    p.m = d->tokens;
    p.n = d->vocab;
    p.k = d->width;
    p.splits = 1;
    p.kb_split = (int)div_up(d->width, TK);
    p.target = d->target;
    p.vocab = d->vocab;
    p.part = part;
    p.tlogit = tlogit;
    if (int st = gemm<false, false, kStats>(x, w, CUtensorMap{}, Matrix{}, p, s)) return st;
  }
  return launch(linear_ce_finish_kernel, div_up(d->tokens, 32), 32 * kFinishWarps, 0, 1, s, part, f.parts, tlogit,
                d->target, d->tokens, d->vocab, d->ignore_index, d->loss, d->lse);
}

extern "C" size_t pdb_linear_ce_bwd_workspace_size(const pdb_linear_ce_bwd_desc* d) {
  if (!d || check(d->tokens, d->vocab, d->width, d->x_stride, d->w_stride, d->dtype) != PDB_OK || d->tokens == 0) return 0;
  return (size_t)plan_bwd(d->tokens, d->vocab, d->width, d->dtype).bytes;
}

extern "C" int pdb_linear_ce_bwd(const pdb_linear_ce_bwd_desc* d, void* stream) {
  if (!d) return set_error(PDB_ERR_ARG, "null descriptor");
  if (int st = check(d->tokens, d->vocab, d->width, d->x_stride, d->w_stride, d->dtype)) return st;
  const int size = d->dtype == PDB_F32 ? 4 : 2;
  if (d->dx && (d->dx_stride < d->width || d->dx_stride * size % 16 != 0 || !a16(d->dx)))
    return set_error(PDB_ERR_ALIGN, "linear cross entropy: dx must be 16-byte aligned with rows of whole 16 bytes");
  if (d->dw && (d->dw_stride < d->width || d->dw_stride * size % 16 != 0 || !a16(d->dw)))
    return set_error(PDB_ERR_ALIGN, "linear cross entropy: dw must be 16-byte aligned with rows of whole 16 bytes");
  if (!d->dx && !d->dw) return set_error(PDB_ERR_ARG, "linear cross entropy: neither dx nor dw");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->tokens == 0) {  // nothing adds to dw
    if (!d->dw) return PDB_OK;
    return cuda_status(cudaMemset2DAsync(d->dw, d->dw_stride * size, 0, d->width * size, d->vocab, s), "linear cross entropy: zero dw");
  }
  if (!d->x || !d->w || !d->target || !d->lse || !d->dloss)
    return set_error(PDB_ERR_ARG, "linear cross entropy: null x / w / target / lse / dloss");
  if (!a16(d->x) || !a16(d->w))
    return set_error(PDB_ERR_ALIGN, "linear cross entropy: x and w must be 16-byte aligned");
  const BwdPlan b = plan_bwd(d->tokens, d->vocab, d->width, d->dtype);
  if (!d->workspace || d->workspace_bytes < (size_t)b.bytes || !a16(d->workspace))
    return set_error(PDB_ERR_ARG, "linear cross entropy: workspace too small or not 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(d->workspace);
  float* dx_acc = reinterpret_cast<float*>(ws + b.dx_acc);
  float* dw_acc = reinterpret_cast<float*>(ws + b.dw_acc);
  float* unit = reinterpret_cast<float*>(ws + b.unit);
  int* state = reinterpret_cast<int*>(ws + b.state);
  int* token_of = reinterpret_cast<int*>(ws + b.token_of);
  const Matrix x{d->x, d->tokens, d->width, d->x_stride}, xp{ws + b.xp, d->tokens, d->width, b.ldp};
  const int64_t* target = reinterpret_cast<const int64_t*>(ws + b.target);
  const float *lse = reinterpret_cast<const float*>(ws + b.lse), *dloss = reinterpret_cast<const float*>(ws + b.dloss);
  if (int st = d->dtype == PDB_F32 ? pack<float>(*d, b, ws, s) : pack<__nv_bfloat16>(*d, b, ws, s)) return st;
  if (d->dtype == PDB_F32) {
    for (int64_t i = 0; i < b.pieces; ++i) {
      const int64_t v0 = i * b.piece, nv = std::min(b.piece, d->vocab - v0);
      const Matrix w{static_cast<const float*>(d->w) + v0 * d->w_stride, nv, d->width, d->w_stride};
      const Matrix g{ws, d->tokens, nv, b.piece};
      F32Args p = f32_product(x, w, d->tokens, nv, d->width);
      p.xp = static_cast<const float*>(xp.p);
      p.ldp = xp.ld;
      p.state = state;
      p.dyn = 1;
      p.target = target;
      p.col0 = v0;
      p.vocab = d->vocab;
      p.lse = lse;
      p.dloss = dloss;
      p.out = reinterpret_cast<float*>(ws);
      p.ldo = b.piece;
      if (int st = f32_gemm<false, false, kDlogits>(p, s)) return st;
      if (d->dw) {
        F32Args q = f32_product(g, x, nv, d->width, d->tokens);
        q.xp = p.xp;
        q.ldp = p.ldp;
        q.state = state;
        q.dyn = 2;
        float* dw = static_cast<float*>(d->dw) + v0 * d->dw_stride;
        q.splits = b.dw_splits;
        q.out = q.splits > 1 ? dw_acc : dw;
        q.ldo = q.splits > 1 ? d->width : d->dw_stride;
        if (int st = f32_gemm<true, true, kOut>(q, s)) return st;
        if (q.splits > 1)
          if (int st = join(dw_acc, q.splits, nv, d->width, nullptr, nullptr, nullptr, dw, d->dw_stride, s)) return st;
      }
      if (d->dx) {
        F32Args q = f32_product(g, w, d->tokens, d->width, nv);
        q.state = state;
        q.dyn = 1;
        q.splits = b.dx_splits;
        q.token_of = q.splits > 1 ? nullptr : token_of;
        q.out = q.splits > 1 ? dx_acc : static_cast<float*>(d->dx);
        q.ldo = q.splits > 1 ? d->width : d->dx_stride;
        q.add = i > 0;
        if (int st = f32_gemm<false, true, kOut>(q, s)) return st;
      }
    }
    if (d->dx && b.dx_splits > 1)
      return join(dx_acc, b.dx_splits, d->tokens, d->width, nullptr, state, token_of, static_cast<float*>(d->dx), d->dx_stride, s);
    return PDB_OK;
  }
  for (int64_t i = 0; i < b.pieces; ++i) {
    const int64_t v0 = i * b.piece, nv = std::min(b.piece, d->vocab - v0);
    const Matrix w{static_cast<const __nv_bfloat16*>(d->w) + v0 * d->w_stride, nv, d->width, d->w_stride};
    const Matrix g{ws, d->tokens, nv, b.piece};
    Args p{};
    p.m = d->tokens;
    p.n = nv;
    p.k = d->width;
    p.splits = 1;
    p.kb_split = (int)div_up(d->width, TK);
    p.state = state;
    p.dyn = 1;
    p.target = target;
    p.col0 = v0;
    p.vocab = d->vocab;
    p.lse = lse;
    p.dloss = dloss;
    p.unit = unit;
    CUtensorMap tc;
    if (int st = map2d(&tc, g, 64, 32)) return st;
    if (int st = gemm<false, false, kDlogits>(x, w, tc, xp, p, s)) return st;
    if (d->dw) {
      Args q{};
      q.m = nv;
      q.n = d->width;
      q.k = d->tokens;
      q.splits = b.dw_splits;
      q.state = state;
      q.dyn = 2;
      q.unit = unit;
      const Matrix dw{static_cast<__nv_bfloat16*>(d->dw) + v0 * d->dw_stride, nv, d->width, d->dw_stride};
      float* acc = b.dw_splits > 1 ? dw_acc : nullptr;
      if (int st = gemm_out<true, true>(g, x, dw, acc, xp, q, s)) return st;
      if (acc)
        if (int st = join<__nv_bfloat16>(acc, q.splits, q.m, q.n, unit, nullptr, nullptr,
                                         static_cast<__nv_bfloat16*>(d->dw) + v0 * d->dw_stride, dw.ld, s))
          return st;
    }
    if (d->dx) {
      Args q{};
      q.m = d->tokens;
      q.n = d->width;
      q.k = nv;
      // every piece takes at most the first one's number of shares, and adds to their sums
      q.kb_split = (int)div_up(div_up(nv, TK), b.dx_splits);
      q.splits = (int)div_up(div_up(nv, TK), q.kb_split);
      q.state = state;
      q.dyn = 1;
      q.token_of = token_of;
      q.unit = unit;
      q.add = i > 0;
      const Matrix dx{d->dx, d->tokens, d->width, d->dx_stride};
      if (int st = gemm_out<false, true>(g, w, dx, b.dx_splits > 1 || b.pieces > 1 ? dx_acc : nullptr, Matrix{}, q, s)) return st;
    }
  }
  if (d->dx && (b.dx_splits > 1 || b.pieces > 1))
    return join(dx_acc, b.dx_splits, d->tokens, d->width, unit, state, token_of, static_cast<__nv_bfloat16*>(d->dx),
                d->dx_stride, s);
  return PDB_OK;
}
