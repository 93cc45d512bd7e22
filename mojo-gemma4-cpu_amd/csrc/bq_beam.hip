// Selection over beams and vocabulary: for each request the n best of
//   score[k] + logit[k, v] - logsumexp(logits[k, :])
// over its beams k and tokens v, ties to the lowest (k, v).  A finished beam has
// one candidate, the end token at its own score.
//
// Bound: every logit is read once, and an exponential in 64 bits is taken of each.
// k_beam_parts reads them: a wave takes kPart values of a row and leaves their
// maximum and the sum of their exponentials above it.  The n best elements lie in the
// n parts with the best maxima (an element of another part has n better elements
// ahead of it, one in each), so k_beam_pick, a workgroup per request, ranks the parts
// and reads n of them again.
//
// Sums and scores are 64 bits: beams are compared across rows, and 32 bits of
// a score near -20 make ties of candidates that are 2e-6 apart.
#include <algorithm>

#include "bq_half.hpp"
#include "bq_kernels.hpp"

namespace bq {

namespace {

constexpr int kPart = 2048;          // logits per part
constexpr int kPickThreads = 1024;
constexpr int kListed = 2048;        // candidates ranked in LDS

struct BeamPart {
  double sum;  // of e^(x - max)
  float max;   // -inf: no candidate
  int32_t pad;
};

// 16 bytes of logits: N values
struct F32In {
  typedef float raw;
  static constexpr int N = 4;
  __device__ static float value(raw r) { return r; }
  __device__ static void unpack(v4u w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  }
};
struct Bf16In {
  typedef uint16_t raw;
  static constexpr int N = 8;
  __device__ static float value(raw r) { return bf16_to_f32(r); }
  __device__ static void unpack(v4u w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = Bf16::lo(w[i]), x[2 * i + 1] = Bf16::hi(w[i]);
  }
};
struct F16In {
  typedef uint16_t raw;
  static constexpr int N = 8;
  __device__ static float value(raw r) { return (float)__builtin_bit_cast(_Float16, r); }
  __device__ static void unpack(v4u w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = F16::lo(w[i]), x[2 * i + 1] = F16::hi(w[i]);
  }
};

// e^(x - m) for x <= m in 64 bits, to 1e-12 of itself: 2^(k / 32) from a table, times
// the series of 2^(f / 32), |f| <= 1/2, to the fourth power (the next term is
// (ln2 / 64)^5 / 120 = 1.3e-12).  The table's 32 values lie in banks of their own, so
// that a wave's look-ups never meet.  x is taken as at least m - 600.
struct Exp64 {
  const double* table;  // LDS, 2^(k / 32)
  double m32;           // -m * 32 / ln 2
  float floor;
  static constexpr double kScale = 46.166241308446829;  // 32 / ln 2
  __device__ Exp64(const double* t, float m)
      : table(t), m32(-(double)m * kScale), floor(m - 600.0f) {}
  __device__ double operator()(float x, double add) const {  // add + e^(x - m)
    const double t = __builtin_fma((double)fmaxf(x, floor), kScale, m32);
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: its low bits are the integer
    const double r = t + magic;
    const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, r);
    const double f = t - (r - magic);
    constexpr double c = 0.021660849392498290;  // ln 2 / 32
    double p = c * c * c * c / 24;
    p = __builtin_fma(p, f, c * c * c / 6);
    p = __builtin_fma(p, f, c * c / 2);
    p = __builtin_fma(p, f, c);
    p = __builtin_fma(p, f, 1.0);
    const uint64_t e = __builtin_bit_cast(uint64_t, table[k & 31]) +
                       ((uint64_t)(uint32_t)((k >> 5) << 20) << 32);
    return __builtin_fma(__builtin_bit_cast(double, e), p, add);
  }
};

__device__ inline void exp64_table(double* lds) {  // by the first 32 threads
  if (threadIdx.x < 32) lds[threadIdx.x] = exp2((double)threadIdx.x / 32);
}

// Part `part` of a row, in 16-byte words from the aligned address at or before the
// row's start: x[i][e] is token first + (i * 64 + lane) * N + e, -inf outside the row.
template <typename In>
struct PartValues {
  static constexpr int WORDS = kPart / (64 * In::N);
  float x[WORDS][In::N];
  int first;
  __device__ void load(const typename In::raw* row, int vocab, int part) {
    const int lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename In::raw));
    first = part * kPart - lead;
    v4u w[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      const int v = first + (i * 64 + lane_id()) * In::N;
      if (v >= 0 && v + In::N <= vocab) w[i] = *reinterpret_cast<const v4u*>(row + v);
    }
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      const int v = first + (i * 64 + lane_id()) * In::N;
      if (v >= 0 && v + In::N <= vocab) {
        In::unpack(w[i], x[i]);
      } else {
#pragma unroll
        for (int e = 0; e < In::N; ++e)
          x[i][e] = v + e >= 0 && v + e < vocab ? In::value(row[v + e]) : -INFINITY;
      }
    }
  }
  __device__ int token(int i, int e) const { return first + (i * 64 + lane_id()) * In::N + e; }
};

template <typename In>
__global__ __launch_bounds__(256) void k_beam_parts(BeamArgs a) {
  __shared__ double table[32];
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t r = w / a.parts;
  const bool on = r < (int64_t)a.batch * a.beams && !(a.finished && a.finished[r]);
  PartValues<In> p;
  if (on)
    p.load(static_cast<const typename In::raw*>(a.logits) + r * a.row_stride, a.vocab,
           (int)(w - r * a.parts));
  exp64_table(table);  // while the logits come
  __syncthreads();
  if (!on) return;
  float m = -INFINITY;  // NaN is no candidate and adds nothing
#pragma unroll
  for (int i = 0; i < p.WORDS; ++i)
#pragma unroll
    for (int e = 0; e < In::N; ++e) m = fmaxf(m, p.x[i][e]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  double s = 0.0;
  if (m > -INFINITY && m < INFINITY) {
    const Exp64 ex(table, m);
#pragma unroll
    for (int i = 0; i < p.WORDS; ++i)
#pragma unroll
      for (int e = 0; e < In::N; ++e) s = ex(p.x[i][e], s);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
  }
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
constexpr Cand kNone{-INFINITY, kNowhere};

struct PickLds {
  double table[32];
  Cand group[64];               // the best of each group of threads
  Cand list[kListed];
  double lse[kMaxBeams], score[kMaxBeams];
  Cand chosen[kMaxPicks];
  Cand bound;
  int part[kMaxPicks];
  int count;
};

// the best of WIDTH neighbouring lanes, in all of them
template <int WIDTH>
__device__ inline Cand lanes_best(Cand c) {
#pragma unroll
  for (int d = 1; d < WIDTH; d <<= 1) {
    const Cand o{__shfl_xor(c.score, d), __shfl_xor(c.at, d)};
    if (before(o, c)) c = o;
  }
  return c;
}

// The n best of the candidates that each(f) calls f with (every thread its own, the
// same at every call), in order, to s.chosen; returns how many there are.  All that
// are no worse than `bound` go to a list in LDS, and each finds its rank by counting
// those before it.  Lists that do not fit (thousands of equal scores) are walked n
// times instead, each time for the best after the last.
template <typename Each>
__device__ inline int pick(PickLds& s, int n, Cand bound, Each&& each) {
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  each([&](const Cand& c) {
    if (c.at == kNowhere || before(bound, c)) return;
    const int k = atomicAdd(&s.count, 1);
    if (k < kListed) s.list[k] = c;
  });
  __syncthreads();
  const int m = s.count;
  if (m <= kListed) {
    for (int i = threadIdx.x; i < m; i += kPickThreads) {
      const Cand c = s.list[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < m; ++j) rank += before(s.list[j], c);
      if (rank < n) s.chosen[rank] = c;
    }
    __syncthreads();
    return min(n, m);
  }
  Cand last{INFINITY, -1};
  int r = 0;
  for (; r < n; ++r) {
    Cand best = kNone;
    each([&](const Cand& c) {
      if (before(last, c) && before(c, best)) best = c;
    });
    best = lanes_best<64>(best);
    if (lane_id() == 0) s.group[threadIdx.x >> 6] = best;
    __syncthreads();
    best = s.group[0];
    for (int w = 1; w < kPickThreads / 64; ++w)
      if (before(s.group[w], best)) best = s.group[w];
    if (threadIdx.x == 0) s.chosen[r] = best;
    __syncthreads();
    if (best.at == kNowhere) break;
    last = best;
  }
  return r;
}

template <typename In>
__global__ __launch_bounds__(kPickThreads) void k_beam_pick(BeamArgs a) {
  __shared__ PickLds s;
  const int b = blockIdx.x, lane = lane_id(), wave = threadIdx.x >> 6;
  const int64_t row0 = (int64_t)b * a.beams;
  const BeamPart* parts = static_cast<const BeamPart*>(a.workspace) + row0 * a.parts;
  exp64_table(s.table);
  __syncthreads();

  for (int k = wave; k < a.beams; k += kPickThreads / 64) {
    double lse = 0.0;
    if (!(a.finished && a.finished[row0 + k])) {
      const BeamPart* p = parts + (int64_t)k * a.parts;
      float m = -INFINITY;
      for (int i = lane; i < a.parts; i += 64) m = fmaxf(m, p[i].max);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
      const Exp64 ex(s.table, m);
      double sum = 0.0;
      for (int i = lane; i < a.parts; i += 64)
        if (p[i].max > -INFINITY) sum = __builtin_fma(p[i].sum, ex(p[i].max, 0.0), sum);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
      lse = m < INFINITY ? (double)m + log(sum) : NAN;  // a row with +inf has no candidates
    }
    if (lane == 0) {
      s.lse[k] = lse;
      s.score[k] = a.scores[row0 + k];
    }
  }
  __syncthreads();

  // the n parts with the best maxima
  const int total = a.beams * a.parts;
  auto each_part = [&](auto&& f) {
    for (int id = threadIdx.x; id < total; id += kPickThreads) {
      const int k = id / a.parts;
      Cand c{-INFINITY, id};
      if (a.finished && a.finished[row0 + k]) {
        if (id == k * a.parts) c.score = s.score[k];
      } else {
        const float m = parts[id].max;
        if (m > -INFINITY) c.score = s.score[k] + ((double)m - s.lse[k]);
      }
      if (c.score > -INFINITY) f(c);
    }
  };
  // What is worse than the n-th best of all groups' best is not among the n best.
  constexpr int lanes = 16, groups = kPickThreads / lanes;
  Cand best = kNone;
  each_part([&](const Cand& c) {
    if (before(c, best)) best = c;
  });
  best = lanes_best<lanes>(best);
  if (lane % lanes == 0) s.group[threadIdx.x / lanes] = best;
  __syncthreads();
  best = s.group[lane];
  int rank = 0;
#pragma unroll 8
  for (int g = 0; g < groups; ++g) rank += before(s.group[g], best);
  if (wave == 0 && best.at != kNowhere && rank == a.n - 1) s.bound = best;
  const bool enough = __popcll(__ballot(best.at != kNowhere)) >= a.n;
  __syncthreads();
  Cand bound = enough ? s.bound : kNone;
  const int picks = pick(s, a.n, bound, each_part);

  // the n best of their elements: no worse than the worst part's best
  for (int q = threadIdx.x; q < picks; q += kPickThreads) s.part[q] = (int)s.chosen[q].at;
  bound = picks < a.n ? kNone : Cand{s.chosen[picks - 1].score, kNowhere - 1};
  __syncthreads();
  auto each_value = [&](auto&& f) {
#pragma unroll 1
    for (int q = wave; q < picks; q += kPickThreads / 64) {
      const int id = s.part[q], k = id / a.parts, part = id - k * a.parts;
      const double sc = s.score[k], lse = s.lse[k];
      if (a.finished && a.finished[row0 + k]) {
        if (lane == 0) f(Cand{sc, (int64_t)k * a.vocab + a.eos_id});
        continue;
      }
      const typename In::raw* row =
          static_cast<const typename In::raw*>(a.logits) + (row0 + k) * a.row_stride;
      PartValues<In> p;
      p.load(row, a.vocab, part);
      uint32_t good = 0;  // few pass: they are read once more
#pragma unroll
      for (int i = 0; i < p.WORDS; ++i)
#pragma unroll
        for (int e = 0; e < In::N; ++e) {
          const double v = sc + ((double)p.x[i][e] - lse);
          good |= (uint32_t)(v >= bound.score && v > -INFINITY) << (i * In::N + e);
        }
      for (; good; good &= good - 1) {
        const int at = __builtin_ctz(good), v = p.token(at / In::N, at % In::N);
        f(Cand{sc + ((double)In::value(row[v]) - lse), (int64_t)k * a.vocab + v});
      }
    }
  };
  const int found = pick(s, a.n, bound, each_value);
  for (int r = threadIdx.x; r < a.n; r += kPickThreads) {
    const int64_t o = (int64_t)b * a.n + r;
    const bool any = r < found;
    const Cand c = any ? s.chosen[r] : kNone;
    const int k = any ? (int)(c.at / a.vocab) : -1;
    const int v = any ? (int)(c.at - (int64_t)k * a.vocab) : -1;
    a.out_scores[o] = any ? (float)c.score : -INFINITY;
    a.out_parents[o] = any ? (int)(row0 + k) : -1;
    a.out_tokens[o] = v;
    if (a.out_finished)
      a.out_finished[o] = any && ((a.finished && a.finished[row0 + k]) || v == a.eos_id);
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

// rows that start off a 16-byte boundary have up to 7 values ahead of their first
int beam_parts(int vocab) { return (vocab + 7 + kPart - 1) / kPart; }
size_t beam_workspace(int64_t rows, int vocab) {
  return (size_t)rows * beam_parts(vocab) * sizeof(BeamPart);
}

hipError_t launch_beam_select(const BeamArgs& a, int dtype_bytes, bool f16, hipStream_t st) {
  if (dtype_bytes == 4) return launch<F32In>(a, st);
  return f16 ? launch<F16In>(a, st) : launch<Bf16In>(a, st);
}

}  // namespace bq
