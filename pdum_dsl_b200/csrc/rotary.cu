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
// fraction of a turn, goes through sincospi.  The error is position * 2^-65 of a
// turn from the table plus f32's on [-1, 1].
//
// HBM-bound: every element is read and written once.  A thread holds the cos and
// sin of one 16-byte group of pairs and turns that group in several heads of its
// position, so the angles cost little.
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
  int half;        // pairs
  int units;       // groups of VEC pairs (halves) or VEC / 2 pairs (interleaved), then of VEC features that pass
  int rot_units;
  int chunk, chunks;  // heads per thread, and how many such shares
  float amplitude;
  uint64_t turns[PDB_ROTARY_MAX_PAIRS];  // per position, in 2^-64 of a turn
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// INTER: a group is VEC features, VEC / 2 pairs (one pair of two accesses where no address is even).
// Else a group is VEC pairs, VEC features from each half.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ Args p) {
  using P = Pack<T, VEC>;
  constexpr int NP = INTER ? (VEC > 1 ? VEC / 2 : 1) : VEC;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int unit = (int)(i % p.units);
  const int64_t rest = i / p.units;
  const int share = (int)(rest % p.chunks);
  const int64_t bt = rest / p.chunks;
  const int64_t b = bt / p.seqlen, t = bt - b * p.seqlen;
  if (b >= p.batch) return;
  const int h0 = share * p.chunk, total = p.heads[0] + p.heads[1];
  const int h1 = h0 + p.chunk < total ? h0 + p.chunk : total;
  const bool turn = unit < p.rot_units;
  const int j0 = unit * NP;
  const int64_t f0 = turn ? (INTER ? 2 * j0 : j0) : (int64_t)2 * p.half + (unit - p.rot_units) * VEC;
  float cs[NP], sn[NP];
  if (turn) {
    const uint64_t pos = (uint64_t)(p.pos ? p.pos[b * p.ps[0] + t * p.ps[1]] : p.start + t);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      // the signed top 32 bits: half turns in units of 2^-31
      const int frac = (int)((pos * p.turns[j0 + j] + 0x80000000ull) >> 32);
      sincospif((float)frac * 4.656612873077393e-10f, &sn[j], &cs[j]);
      sn[j] *= p.amplitude;
      cs[j] *= p.amplitude;
    }
  }
  for (int h = h0; h < h1; ++h) {
    const int w = h >= p.heads[0];
    const int64_t hh = w ? h - p.heads[0] : h;
    const T* x = static_cast<const T*>(p.x[w]) + b * p.xs[w][0] + hh * p.xs[w][1] + t * p.xs[w][2] + f0;
    T* y = static_cast<T*>(p.y[w]) + b * p.ys[w][0] + hh * p.ys[w][1] + t * p.ys[w][2] + f0;
    P u = *reinterpret_cast<const P*>(x);
    if (turn) {
      if constexpr (INTER && VEC == 1) {
        const float a = to_f32(u.v[0]), c = to_f32(x[1]);
        from_f32(u.v[0], a * cs[0] - c * sn[0]);
        from_f32(y[1], c * cs[0] + a * sn[0]);
      } else if constexpr (INTER) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float a = to_f32(u.v[2 * j]), c = to_f32(u.v[2 * j + 1]);
          from_f32(u.v[2 * j], a * cs[j] - c * sn[j]);
          from_f32(u.v[2 * j + 1], c * cs[j] + a * sn[j]);
        }
      } else {
        P v = *reinterpret_cast<const P*>(x + p.half);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float a = to_f32(u.v[j]), c = to_f32(v.v[j]);
          from_f32(u.v[j], a * cs[j] - c * sn[j]);
          from_f32(v.v[j], c * cs[j] + a * sn[j]);
        }
        *reinterpret_cast<P*>(y + p.half) = v;
      }
    }
    *reinterpret_cast<P*>(y) = u;
  }
}

template <typename T, int VEC>
int launch(Args& p, const pdb_rotary_desc& d, cudaStream_t s) {
  const bool inter = d.interleaved != 0;
  p.rot_units = inter && VEC > 1 ? (int)(d.rotary_dim / VEC) : p.half / VEC;
  // in place there is nothing to do for the features that pass through
  const bool copy = (p.heads[0] && p.x[0] != p.y[0]) || (p.heads[1] && p.x[1] != p.y[1]);
  p.units = p.rot_units + (copy ? (int)((d.head_dim - d.rotary_dim) / VEC) : 0);
  if (p.units == 0) return PDB_OK;
  int dev = 0;
  cudaGetDevice(&dev);
  const int total = p.heads[0] + p.heads[1];
  const int64_t points = p.batch * p.seqlen * p.units;
  // heads per thread: 8 where that leaves every SM four blocks, fewer otherwise
  const int64_t want = (int64_t)sm_count(dev) * 4 * kThreads;
  p.chunk = 8;
  while (p.chunk > 1 && points * ((total + p.chunk - 1) / p.chunk) < want) p.chunk >>= 1;
  p.chunks = (total + p.chunk - 1) / p.chunk;
  const int64_t blocks = (points * p.chunks + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) return set_error(PDB_ERR_SHAPE, "rotary: too many heads and positions for one launch");
  if (inter)
    rotary_kernel<T, VEC, true><<<(unsigned)blocks, kThreads, 0, s>>>(p);
  else
    rotary_kernel<T, VEC, false><<<(unsigned)blocks, kThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "rotary launch");
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
  fit(inter ? d->rotary_dim : p.half);
  fit(d->head_dim - d->rotary_dim);
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
      }
    }
  }
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
    const uint64_t turns = (uint64_t)std::ldexp(per - std::floor(per), 64);
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
