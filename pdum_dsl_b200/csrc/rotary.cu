// Rotary positions: pairs of features of a head turn by an angle that grows with
// the position, and its gradient, the inverse turn.
//
//   a' = (a cos - b sin) m     b' = (b cos + a sin) m     angle = position * inv_freq[j]
//
// over the pairs (a, b) = (x[j], x[r/2 + j]) (halves) or (x[2j], x[2j+1])
// (interleaved), j < r/2; the features from r on pass through.  m is an
// amplitude that scalings for long contexts put on cos and sin.
//
// Angles.  position * inv_freq in f32 has no digits left at far positions (an
// error of 0.06 rad at position 10^6).  Here a frequency is a fraction of a turn
// per position in 64-bit fixed point: the integer product position * turns mod
// 2^64 drops whole turns exactly, for any int64 position, and what is left, the
// fraction of a turn, goes through sincospi.  What remains is the table's own
// error, times the position: |inv_freq| / 2 pi in f64 (the division and the
// constant, together 2^-52 of the frequency at most) cut to 2^-64 of a turn, so an
// angle is off by |position| (2^-52 |inv_freq| + 2^-61) radians, about what the
// product position * inv_freq would lose in f64, and by f32's on [-1, 1].
//
// HBM-bound: every element is read and written once.  A thread holds the cos and
// sin of one 16-byte group of pairs and turns that group in several heads of its
// position, so the angles cost little; the loads of four heads are in flight before
// the first is turned, and the turns run on two pairs per instruction.  On a B200,
// 8 x 4096 positions of 32 + 8 heads of 128 bf16: 105 us, 6.4 TB/s.
#include <cmath>

#include "common.cuh"

namespace pdb {
namespace {

constexpr int kThreads = 256;

struct Args {
  const void* x[2];
  void* y[2];
  int64_t xs[2][3], ys[2][3];  // (batch, head, row)
  int heads[2];                // of x[0] and x[1]; heads[1] may be 0
  const int64_t* pos;
  int64_t ps[2], start;
  int64_t batch, seqlen;
  int half;       // pairs
  int units;      // groups of VEC pairs (halves) or VEC / 2 pairs (interleaved), then of VEC features that pass
  int rot_units;
  int64_t pass0;  // the first feature of the groups that pass
  int per_block;  // positions that a block's threads cover
  int chunk;      // heads per thread
  int shares0;    // shares of x[0]'s heads; x[1]'s follow
  float amplitude;
  alignas(16) uint64_t turns[PDB_ROTARY_MAX_PAIRS];  // per position, in 2^-64 of a turn
};

// N entries of the table.  Through the constant port, lanes that want different entries are served one after another,
// which narrow groups (up to 32 different entries in a warp) take by a generic load instead.
template <int N>
__device__ __forceinline__ void load_turns(const uint64_t* at, uint64_t (&v)[N]) {
  if constexpr (N == 1) {
    asm("ld.b64 %0, [%1];" : "=l"(v[0]) : "l"(at));
  } else if constexpr (N == 2) {
    asm("ld.v2.b64 {%0, %1}, [%2];" : "=l"(v[0]), "=l"(v[1]) : "l"(at));
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = at[j];
  }
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// VEC elements as f32 and back, two at a time where there are two.
template <typename T, int VEC>
__device__ __forceinline__ void widen(const Pack<T, VEC>& u, float (&f)[VEC]) {
  if constexpr (sizeof(T) == 2 && VEC > 1) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {  // a bf16 is the upper half of its f32
      f[2 * j] = __uint_as_float(w[j] << 16);
      f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = to_f32(u.v[j]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void narrow(const float (&f)[VEC], Pack<T, VEC>& u) {
  if constexpr (sizeof(T) == 2 && VEC > 1) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) w[j] = pack_bf16(f[2 * j], f[2 * j + 1]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) from_f32(u.v[j], f[j]);
  }
}
// (a, c) -> (a cs - c sn, c cs + a sn) for N pairs
template <int N>
__device__ __forceinline__ void turn_pairs(float (&a)[N], float (&c)[N], const float (&cs)[N], const float (&sn)[N]) {
  if constexpr (N == 1) {
    const float t = a[0] * cs[0] - c[0] * sn[0];
    c[0] = c[0] * cs[0] + a[0] * sn[0];
    a[0] = t;
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const uint64_t x = f2_pack(a[j], a[j + 1]), y = f2_pack(c[j], c[j + 1]), u = f2_pack(cs[j], cs[j + 1]);
      f2_unpack(f2_fma(x, u, f2_mul(y, f2_pack(-sn[j], -sn[j + 1]))), a[j], a[j + 1]);
      f2_unpack(f2_fma(y, u, f2_mul(x, f2_pack(sn[j], sn[j + 1]))), c[j], c[j + 1]);
    }
  }
}

// INTER: a group is VEC features, VEC / 2 pairs (one pair of two accesses where no address is even); the last group that
// turns may reach into the features that pass.  Else a group is VEC pairs, VEC features from each half.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ Args p) {
  using P = Pack<T, VEC>;
  constexpr int NP = INTER ? (VEC > 1 ? VEC / 2 : 1) : VEC, FLIGHT = 4;
  // the second access of a group, where it has one: the other half's, or the other feature of a lone pair
  constexpr bool TWO = !INTER || VEC == 1;
  const int span = p.units < kThreads ? p.units : kThreads;
  const int unit = blockIdx.z * kThreads + (int)threadIdx.x % span, at = (int)threadIdx.x / span;
  const int64_t bt = (int64_t)blockIdx.x * p.per_block + at, points = p.batch * p.seqlen;
  if (at >= p.per_block || unit >= p.units || bt >= points) return;
  int64_t b, t;
  if ((uint64_t)points <= 0xffffffffu) {
    b = (uint32_t)bt / (uint32_t)p.seqlen;
    t = (uint32_t)bt % (uint32_t)p.seqlen;
  } else {
    b = bt / p.seqlen;
    t = bt % p.seqlen;
  }
  // this block's share of the heads of one of the tensors
  const int w = blockIdx.y >= p.shares0;
  const int h0 = (blockIdx.y - (w ? p.shares0 : 0)) * p.chunk, n = min(p.chunk, p.heads[w] - h0);
  const bool turn = unit < p.rot_units;
  const int j0 = unit * NP;
  const int64_t f0 = turn ? (INTER ? 2 * j0 : j0) : p.pass0 + (int64_t)(unit - p.rot_units) * VEC;
  const int other = INTER ? 1 : p.half;
  float cs[NP], sn[NP];
  if (turn) {
    const uint64_t pos = (uint64_t)(p.pos ? p.pos[b * p.ps[0] + t * p.ps[1]] : p.start + t);
    uint64_t turns[NP];
    load_turns<NP>(p.turns + j0, turns);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      // the signed top 32 bits: half turns in units of 2^-31
      const int frac = (int)((pos * turns[j] + 0x80000000ull) >> 32);
      sincospif((float)frac * 4.656612873077393e-10f, &sn[j], &cs[j]);
      sn[j] *= p.amplitude;
      cs[j] *= p.amplitude;
    }
  }
  const int64_t xh = p.xs[w][1], yh = p.ys[w][1];
  const T* x = static_cast<const T*>(p.x[w]) + b * p.xs[w][0] + h0 * xh + t * p.xs[w][2] + f0;
  T* y = static_cast<T*>(p.y[w]) + b * p.ys[w][0] + h0 * yh + t * p.ys[w][2] + f0;
  for (int h = 0; h < n; h += FLIGHT) {
    P u[FLIGHT], v[FLIGHT];
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i, x += xh) {
      if (h + i >= n) break;
      u[i] = *reinterpret_cast<const P*>(x);
      if (TWO && turn) v[i] = *reinterpret_cast<const P*>(x + other);
    }
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i, y += yh) {
      if (h + i >= n) break;
      if (turn) {
        float f[VEC];
        widen<T, VEC>(u[i], f);
        if constexpr (TWO) {
          float g[VEC];
          widen<T, VEC>(v[i], g);
          turn_pairs<NP>(f, g, cs, sn);
          narrow<T, VEC>(g, v[i]);
          narrow<T, VEC>(f, u[i]);
          *reinterpret_cast<P*>(y + other) = v[i];
        } else {
          const P as_it_was = u[i];
          float a[NP], c[NP];
#pragma unroll
          for (int j = 0; j < NP; ++j) a[j] = f[2 * j], c[j] = f[2 * j + 1];
          turn_pairs<NP>(a, c, cs, sn);
#pragma unroll
          for (int j = 0; j < NP; ++j) f[2 * j] = a[j], f[2 * j + 1] = c[j];
          narrow<T, VEC>(f, u[i]);
          if (j0 + NP > p.half) {
#pragma unroll
            for (int j = 0; j < NP; ++j)
              if (j0 + j >= p.half) u[i].v[2 * j] = as_it_was.v[2 * j], u[i].v[2 * j + 1] = as_it_was.v[2 * j + 1];
          }
        }
      }
      *reinterpret_cast<P*>(y) = u[i];
    }
  }
}

template <typename T, int VEC, bool INTER>
int launch(Args& p, const pdb_rotary_desc& d, cudaStream_t s) {
  constexpr int NP = INTER ? (VEC > 1 ? VEC / 2 : 1) : VEC, G = INTER ? 2 * NP : VEC;
  p.rot_units = INTER ? (p.half + NP - 1) / NP : p.half / VEC;
  p.pass0 = INTER ? (int64_t)p.rot_units * G : 2 * (int64_t)p.half;
  // in place there is nothing to do for the features that pass through
  const bool copy = (p.heads[0] && p.x[0] != p.y[0]) || (p.heads[1] && p.x[1] != p.y[1]);
  p.units = p.rot_units + (copy ? (int)((d.head_dim - p.pass0) / VEC) : 0);
  if (p.units == 0) return PDB_OK;
  int dev = 0;
  cudaGetDevice(&dev);
  const int span = p.units < kThreads ? p.units : kThreads;
  p.per_block = kThreads / span;
  const int64_t points = p.batch * p.seqlen, least = (int64_t)sm_count(dev) * 4;  // four blocks per SM
  const int64_t bx = (points + p.per_block - 1) / p.per_block;
  const int64_t bz = (p.units + kThreads - 1) / kThreads;
  // heads per thread: 8 (16 of narrow groups, whose angles weigh more) where that leaves every SM four blocks, fewer
  // otherwise
  auto shares = [&](int n) { return (n + p.chunk - 1) / p.chunk; };
  p.chunk = VEC * sizeof(T) >= 8 ? 8 : 16;
  while (p.chunk > 1 && bx * bz * (shares(p.heads[0]) + shares(p.heads[1])) < least) p.chunk >>= 1;
  while (shares(p.heads[0]) + shares(p.heads[1]) > 65535) p.chunk *= 2;
  p.shares0 = shares(p.heads[0]);
  if (bx > 0x7fffffffLL) return set_error(PDB_ERR_SHAPE, "rotary: too many positions for one launch");
  const dim3 grid((unsigned)bx, (unsigned)(p.shares0 + shares(p.heads[1])), (unsigned)bz);
  rotary_kernel<T, VEC, INTER><<<grid, kThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "rotary launch");
}

template <typename T, int VEC>
int launch(Args& p, const pdb_rotary_desc& d, cudaStream_t s) {
  return d.interleaved ? launch<T, VEC, true>(p, d, s) : launch<T, VEC, false>(p, d, s);
}

}  // namespace
}  // namespace pdb

using namespace pdb;

extern "C" int pdb_rotary(const pdb_rotary_desc* d, void* stream) {
  if (!d) return set_error(PDB_ERR_ARG, "null descriptor");
  if (d->batch < 0 || d->seqlen < 0 || d->head_dim < 0 || d->heads[0] < 0 || d->heads[1] < 0)
    return set_error(PDB_ERR_SHAPE, "rotary: negative size");
  if (d->rotary_dim < 0 || d->rotary_dim % 2 != 0 || d->rotary_dim > d->head_dim ||
      d->rotary_dim > 2 * PDB_ROTARY_MAX_PAIRS)
    return set_error(PDB_ERR_SHAPE, "rotary: rotary_dim must be even, at most head_dim and at most %d",
                     2 * PDB_ROTARY_MAX_PAIRS);
  if (d->dtype != PDB_F32 && d->dtype != PDB_BF16)
    return set_error(PDB_ERR_UNSUPPORTED, "rotary: unknown dtype %d", d->dtype);
  if (d->head_dim > (1 << 20) || d->heads[0] + d->heads[1] > (1 << 20))
    return set_error(PDB_ERR_SHAPE, "rotary: head_dim and heads are at most 2^20");
  if (d->batch == 0 || d->seqlen == 0 || d->head_dim == 0 || d->heads[0] + d->heads[1] == 0) return PDB_OK;
  if (d->seqlen > (int64_t(1) << 40) / d->batch) return set_error(PDB_ERR_SHAPE, "rotary: too many positions");
  const int size = d->dtype == PDB_F32 ? 4 : 2;
  Args p{};
  // the widest access that every address, stride and group boundary allows
  int vec = 16 / size;
  const bool inter = d->interleaved != 0;
  p.half = (int)(d->rotary_dim / 2);
  auto fit = [&](int64_t elements) {
    while (vec > 1 && elements % vec != 0) vec >>= 1;
  };
  if (inter) {
    fit(d->head_dim);
  } else {
    fit(p.half);
    fit(d->head_dim - d->rotary_dim);
  }
  for (int w = 0; w < 2; ++w) {
    p.heads[w] = (int)d->heads[w];
    if (d->heads[w] == 0) continue;
    if (!d->x[w] || !d->y[w]) return set_error(PDB_ERR_ARG, "rotary: null x / y");
    if ((reinterpret_cast<uintptr_t>(d->x[w]) | reinterpret_cast<uintptr_t>(d->y[w])) % size != 0)
      return set_error(PDB_ERR_ALIGN, "rotary: x / y not aligned to their type");
    p.x[w] = d->x[w];
    p.y[w] = d->y[w];
    fit((int64_t)(reinterpret_cast<uintptr_t>(d->x[w]) / size));
    fit((int64_t)(reinterpret_cast<uintptr_t>(d->y[w]) / size));
    const int64_t dims[3] = {d->batch, d->heads[w], d->seqlen};
    for (int k = 0; k < 3; ++k) {
      p.xs[w][k] = d->x_stride[w][k];
      p.ys[w][k] = d->y_stride[w][k];
      if (dims[k] > 1) {
        fit(p.xs[w][k]);
        fit(p.ys[w][k]);
        if (p.x[w] == p.y[w] && p.xs[w][k] != p.ys[w][k])
          return set_error(PDB_ERR_ARG, "rotary: a tensor turned in place has one set of strides");
      }
    }
  }
  // threads read and write in no order between heads: a result that starts where another tensor does is a mistake
  if (p.heads[0] && p.heads[1] && (p.y[0] == p.y[1] || p.y[0] == p.x[1] || p.y[1] == p.x[0]))
    return set_error(PDB_ERR_ARG, "rotary: a result overlaps the other tensor");
  p.pos = d->positions;
  p.ps[0] = d->pos_stride[0];
  p.ps[1] = d->pos_stride[1];
  p.start = d->start;
  p.batch = d->batch;
  p.seqlen = d->seqlen;
  p.amplitude = (float)d->amplitude;
  for (int j = 0; j < p.half; ++j) {
    const double f = d->inv_freq[j], per = std::fabs(f) / 6.283185307179586476925286766559;  // turns per position
    if (!(per < 1e9)) return set_error(PDB_ERR_ARG, "rotary: inv_freq[%d] is not a usable frequency", j);
    // whole turns per position change nothing; a backward turn is the negated integer
    const uint64_t turns = (uint64_t)((per - (double)(int64_t)per) * 0x1p64);
    p.turns[j] = (f < 0) != (d->inverse != 0) ? 0 - turns : turns;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->dtype == PDB_F32) {
    switch (vec) {
      case 4: return launch<float, 4>(p, *d, s);
      case 2: return launch<float, 2>(p, *d, s);
      default: return launch<float, 1>(p, *d, s);
    }
  }
  switch (vec) {
    case 8: return launch<__nv_bfloat16, 8>(p, *d, s);
    case 4: return launch<__nv_bfloat16, 4>(p, *d, s);
    case 2: return launch<__nv_bfloat16, 2>(p, *d, s);
    default: return launch<__nv_bfloat16, 1>(p, *d, s);
  }
}
