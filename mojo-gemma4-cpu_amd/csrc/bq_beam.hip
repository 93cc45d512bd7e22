// Selection over beams and vocabulary: for each request the n best of
//   score[k] + logit[k, v] - logsumexp(logits[k, :])
// over its beams k and tokens v, ties to the lowest (k, v).  A finished beam has
// one candidate, the end token at its own score.
//
// Bound: every logit is read once.  k_beam_parts reads them: a wave takes kPart
// values of a row and leaves their maximum and the sum of their exponentials above
// it.  The n best elements lie in the n parts with the best maxima (an element of
// another part has n better elements ahead of it, one in each), so k_beam_pick, a
// workgroup per request, ranks the parts and reads n of them again.
//
// Sums and scores are 64 bits: beams are compared across rows, and 32 bits of
// a score near -20 make ties of candidates that are 2e-6 apart.
#include <algorithm>

#include "bq_half.hpp"
#include "bq_kernels.hpp"

namespace bq {

namespace {

constexpr int kPart = 1024;          // logits per part
constexpr int kPickThreads = 1024;

struct BeamPart {
  double sum;  // of e^(x - max)
  float max;   // -inf: no candidate
  int32_t pad;
};

struct F32In {
  typedef float raw;
  __device__ static float value(raw r) { return r; }
};
struct Bf16In {
  typedef uint16_t raw;
  __device__ static float value(raw r) { return bf16_to_f32(r); }
};
struct F16In {
  typedef uint16_t raw;
  __device__ static float value(raw r) { return (float)__builtin_bit_cast(_Float16, r); }
};

// e^d for d <= 0 in 64 bits, to 1e-11 of itself: 2^n 2^f with |f| <= 1/2, the
// latter's series to the ninth power (the next term is 7e-12)
__device__ inline double exp64(double d) {
  const double t = d * 1.4426950408889634;
  const double n = __builtin_rint(t);
  const double y = (t - n) * 0.6931471805599453;
  double p = 1.0 / 362880;
  p = __builtin_fma(p, y, 1.0 / 40320);
  p = __builtin_fma(p, y, 1.0 / 5040);
  p = __builtin_fma(p, y, 1.0 / 720);
  p = __builtin_fma(p, y, 1.0 / 120);
  p = __builtin_fma(p, y, 1.0 / 24);
  p = __builtin_fma(p, y, 1.0 / 6);
  p = __builtin_fma(p, y, 0.5);
  p = __builtin_fma(p, y, 1.0);
  p = __builtin_fma(p, y, 1.0);
  return n < -1000.0 ? 0.0 : __builtin_ldexp(p, (int)n);
}

__device__ inline double shfl_xor_f64(double v, int d) { return __shfl_xor(v, d); }

// the logits of part `part` of a row: value e * 64 + lane
template <typename In>
__device__ inline void load_part(const typename In::raw* row, int vocab, int part, float (&x)[kPart / 64]) {
#pragma unroll
  for (int e = 0; e < kPart / 64; ++e) {
    const int v = part * kPart + e * 64 + lane_id();
    const float y = v < vocab ? In::value(row[v]) : -INFINITY;
    x[e] = y == y ? y : -INFINITY;  // NaN is no candidate and adds nothing
  }
}

template <typename In>
__global__ __launch_bounds__(256) void k_beam_parts(BeamArgs a) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t r = w / a.parts;
  if (r >= (int64_t)a.batch * a.beams) return;
  const int part = (int)(w - r * a.parts);
  if (a.finished && a.finished[r]) return;
  const typename In::raw* row =
      static_cast<const typename In::raw*>(a.logits) + r * a.row_stride;
  float x[kPart / 64];
  load_part<In>(row, a.vocab, part, x);
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < kPart / 64; ++e) m = fmaxf(m, x[e]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  double s = 0.0;
  if (m > -INFINITY) {
#pragma unroll
    for (int e = 0; e < kPart / 64; ++e)
      if (x[e] > -INFINITY) s += exp64((double)x[e] - (double)m);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) s += shfl_xor_f64(s, d);
  if (lane_id() == 0) static_cast<BeamPart*>(a.workspace)[w] = BeamPart{s, m, 0};
}

// a candidate: a better score first, then a lower place (beam, part or token)
struct Cand {
  double score;
  int64_t at;
};
__device__ inline bool before(const Cand& a, const Cand& b) {
  return a.score > b.score || (a.score == b.score && a.at < b.at);
}
constexpr int64_t kNowhere = INT64_MAX;

// the best candidate of the workgroup, in every thread
__device__ inline Cand block_best(Cand c, Cand* lds) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const Cand o{__shfl_xor(c.score, d), __shfl_xor(c.at, d)};
    if (before(o, c)) c = o;
  }
  if (lane_id() == 0) lds[threadIdx.x >> 6] = c;
  __syncthreads();
  Cand best = lds[0];
  for (int w = 1; w < kPickThreads / 64; ++w)
    if (before(lds[w], best)) best = lds[w];
  __syncthreads();
  return best;
}

template <typename In>
__global__ __launch_bounds__(kPickThreads) void k_beam_pick(BeamArgs a) {
  __shared__ Cand red[kPickThreads / 64];
  __shared__ double base[kMaxBeams];  // score - logsumexp of each beam
  __shared__ int64_t chosen[kMaxPicks];
  const int b = blockIdx.x, lane = lane_id(), wave = threadIdx.x >> 6;
  const int64_t row0 = (int64_t)b * a.beams;
  const BeamPart* parts = static_cast<const BeamPart*>(a.workspace) + row0 * a.parts;

  for (int k = wave; k < a.beams; k += kPickThreads / 64) {
    double lse = 0.0;
    if (!(a.finished && a.finished[row0 + k])) {
      const BeamPart* p = parts + (int64_t)k * a.parts;
      float m = -INFINITY;
      for (int i = lane; i < a.parts; i += 64) m = fmaxf(m, p[i].max);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
      double s = 0.0;
      for (int i = lane; i < a.parts; i += 64)
        if (p[i].max > -INFINITY) s += p[i].sum * exp64((double)p[i].max - (double)m);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) s += shfl_xor_f64(s, d);
      lse = (double)m + log(s);
    }
    if (lane == 0) base[k] = lse;
  }
  __syncthreads();

  const int total = a.beams * a.parts;
  auto part_key = [&](int id) {
    const int k = id / a.parts;
    const double sc = a.scores[row0 + k];
    Cand c{-INFINITY, id};
    if (a.finished && a.finished[row0 + k]) {
      if (id == k * a.parts) c.score = sc;
    } else {
      const float m = parts[id].max;
      if (m > -INFINITY) c.score = sc + ((double)m - base[k]);
    }
    if (!(c.score > -INFINITY)) c = Cand{-INFINITY, kNowhere};
    return c;
  };
  int picks = 0;
  Cand last{INFINITY, -1};
  for (; picks < a.n; ++picks) {
    Cand best{-INFINITY, kNowhere};
    for (int id = threadIdx.x; id < total; id += kPickThreads) {
      const Cand c = part_key(id);
      if (before(last, c) && before(c, best)) best = c;
    }
    best = block_best(best, red);
    if (best.at == kNowhere) break;
    if (threadIdx.x == 0) chosen[picks] = best.at;
    last = best;
  }
  __syncthreads();

  last = Cand{INFINITY, -1};
  for (int r = 0; r < a.n; ++r) {
    Cand best{-INFINITY, kNowhere};
    for (int q = wave; q < picks; q += kPickThreads / 64) {
      const int id = (int)chosen[q], k = id / a.parts, part = id % a.parts;
      const double sc = a.scores[row0 + k];
      if (a.finished && a.finished[row0 + k]) {
        const Cand c{sc, (int64_t)k * a.vocab + a.eos_id};
        if (before(last, c) && before(c, best)) best = c;
        continue;
      }
      const typename In::raw* row =
          static_cast<const typename In::raw*>(a.logits) + (row0 + k) * a.row_stride;
      float x[kPart / 64];
      load_part<In>(row, a.vocab, part, x);
#pragma unroll
      for (int e = 0; e < kPart / 64; ++e) {
        const Cand c{sc + ((double)x[e] - base[k]),
                     (int64_t)k * a.vocab + part * kPart + e * 64 + lane};
        if (c.score > -INFINITY && before(last, c) && before(c, best)) best = c;
      }
    }
    best = block_best(best, red);
    if (threadIdx.x == 0) {
      const int64_t o = (int64_t)b * a.n + r;
      const bool any = best.at != kNowhere;
      const int k = any ? (int)(best.at / a.vocab) : -1;
      const int v = any ? (int)(best.at - (int64_t)k * a.vocab) : -1;
      a.out_scores[o] = any ? (float)best.score : -INFINITY;
      a.out_parents[o] = any ? (int)(row0 + k) : -1;
      a.out_tokens[o] = v;
      if (a.out_finished)
        a.out_finished[o] = any && ((a.finished && a.finished[row0 + k]) || v == a.eos_id);
    }
    last = best;
  }
}

template <typename In>
hipError_t launch(const BeamArgs& a, hipStream_t st) {
  const int64_t waves = (int64_t)a.batch * a.beams * a.parts;
  if ((waves + 3) / 4 > INT32_MAX) return hipErrorInvalidValue;
  k_beam_parts<In><<<(int)((waves + 3) / 4), 256, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  k_beam_pick<In><<<a.batch, kPickThreads, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

int beam_parts(int vocab) { return (vocab + kPart - 1) / kPart; }
size_t beam_workspace(int64_t rows, int vocab) {
  return (size_t)rows * beam_parts(vocab) * sizeof(BeamPart);
}

hipError_t launch_beam_select(const BeamArgs& a, int dtype_bytes, bool f16, hipStream_t st) {
  if (dtype_bytes == 4) return launch<F32In>(a, st);
  return f16 ? launch<F16In>(a, st) : launch<Bf16In>(a, st);
}

}  // namespace bq
