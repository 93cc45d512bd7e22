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
// 256 rows of 262144 f32 logits, a fifth of the beams ended: parts 43 us, 5.0 TB/s of what
// is read, pick 11; 16-bit logits are bound by the exponentials (17 instructions each).
//
// Sums and scores are 64 bits: beams are compared across rows, and 32 bits of
// a score near -20 make ties of candidates that are 2e-6 apart.
#include <algorithm>

#include "bq_half.hpp"
#include "bq_kernels.hpp"

namespace bq {

namespace {

constexpr int kPart = 2048, kSmallPart = 512;  // logits per part
constexpr int kPickThreads = 1024, kWaves = kPickThreads / 64;
constexpr int kListed = 1024;        // candidates ranked in LDS
constexpr int kFusedParts = 2112;    // parts of a request that one launch does all of

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
template <typename In, int PART>
struct PartValues {
  static constexpr int WORDS = PART / (64 * In::N);
  float x[WORDS][In::N];
  int first;
  __device__ void load(const typename In::raw* row, int vocab, int part) {
    const int lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename In::raw));
    first = part * PART - lead;
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

// the maximum of a part and its exponentials' sum, in lane 0
template <typename In, int PART>
__device__ inline BeamPart sum_part(const PartValues<In, PART>& p, const double* table) {
  float m = -INFINITY;  // NaN is no candidate and adds nothing
#pragma unroll
  for (int i = 0; i < p.WORDS; ++i)
#pragma unroll
    for (int e = 0; e < In::N; ++e) m = fmaxf(m, p.x[i][e]);
  m = wave_all_max(m);
  double s = 0.0;
  if (m > -INFINITY && m < INFINITY) {
    const Exp64 ex(table, m);
#pragma unroll
    for (int i = 0; i < p.WORDS; ++i)
#pragma unroll
      for (int e = 0; e < In::N; ++e) s = ex(p.x[i][e], s);
    s = wave_all_sum(s);
  }
  return BeamPart{s, m, 0};
}

template <typename In>
__global__ __launch_bounds__(256) void k_beam_parts(BeamArgs a) {
  __shared__ double table[32];
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t r = w / a.parts;
  const bool on = r < (int64_t)a.batch * a.beams && !(a.finished && a.finished[r]);
  PartValues<In, kPart> p;
  if (on)
    p.load(static_cast<const typename In::raw*>(a.logits) + r * a.row_stride, a.vocab,
           (int)(w - r * a.parts));
  exp64_table(table);  // while the logits come
  __syncthreads();
  if (!on) return;
  const BeamPart part = sum_part(p, table);
  if (lane_id() == 0) static_cast<BeamPart*>(a.workspace)[w] = part;
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
  BeamPart parts[kFusedParts];  // FUSED: the request's
  Cand group[kWaves];           // the best of each wave
  float top[kPickThreads / 4];  // of each four threads
  float wave_top[kWaves];
  int rank[64];
  Cand list[kListed];
  double lse[kMaxBeams], score[kMaxBeams];
  Cand chosen[kMaxPicks];
  float bound;
  int64_t part[kMaxPicks];
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
    // 64 candidates at a time, 16 threads each
    for (int i0 = 0; i0 < m; i0 += 64) {
      const int i = i0 + (threadIdx.x & 63);
      if (threadIdx.x < 64) s.rank[threadIdx.x] = 0;
      __syncthreads();
      if (i < m) {
        const Cand c = s.list[i];
        int rank = 0;
        for (int j = threadIdx.x >> 6; j < m; j += kWaves) rank += before(s.list[j], c);
        if (rank) atomicAdd(&s.rank[threadIdx.x & 63], rank);
      }
      __syncthreads();
      if (threadIdx.x < 64 && i < m && s.rank[threadIdx.x] < n)
        s.chosen[s.rank[threadIdx.x]] = s.list[i];
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
    for (int w = 1; w < kWaves; ++w)
      if (before(s.group[w], best)) best = s.group[w];
    if (threadIdx.x == 0) s.chosen[r] = best;
    __syncthreads();
    if (best.at == kNowhere) break;
    last = best;
  }
  return r;
}

// The largest value of 16 bits that at least n of a wave's values reach (each lane brings
// VALUES of them): from the first bit of their ordered form on.
template <int VALUES>
__device__ inline float nth_of_wave(const float (&v)[VALUES], int n) {
  uint32_t key[VALUES];
#pragma unroll
  for (int i = 0; i < VALUES; ++i) {
    const uint32_t w = __float_as_uint(v[i]);
    key[i] = (int)w < 0 ? ~w : w | 0x80000000u;
  }
  uint32_t nth = 0;
  for (uint32_t bit = 0x80000000u; bit > 0x8000u; bit >>= 1) {
    int reach = 0;
#pragma unroll
    for (int i = 0; i < VALUES; ++i) reach += __popcll(__ballot(key[i] >= (nth | bit)));
    if (reach >= n) nth |= bit;
  }
  if (nth < 0x00800000u) return -INFINITY;  // of which 16 bits would be a NaN's
  return __uint_as_float(nth & 0x80000000u ? nth & 0x7FFFFFFFu : ~nth);
}

// A bound that at least n candidates are no worse than, from the best of each thread's
// (rounded down to 32 bits; -inf: none): the n-th of the best of every four threads;
// where fewer than n of those have any, the best wave's n-th thread.
__device__ inline float nth_of_tops(PickLds& s, float top, int n) {
  float four = fmaxf(top, __shfl_xor(top, 1));
  four = fmaxf(four, __shfl_xor(four, 2));
  if (threadIdx.x % 4 == 0) s.top[threadIdx.x / 4] = four;
  __syncthreads();
  if (threadIdx.x < 64) {
    float v[kPickThreads / 256];
#pragma unroll
    for (int i = 0; i < kPickThreads / 256; ++i) v[i] = s.top[i * 64 + threadIdx.x];
    const float nth = nth_of_wave(v, n);
    if (threadIdx.x == 0) s.bound = nth;
  }
  __syncthreads();
  float bound = s.bound;
  if (bound == -INFINITY) {
    const float mine[1] = {top};
    const float nth = nth_of_wave(mine, n);
    if (lane_id() == 0) s.wave_top[threadIdx.x >> 6] = nth;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) bound = fmaxf(bound, s.wave_top[w]);
  }
  return bound;
}

// FUSED: the parts too, one a wave; the request's last workgroup picks.
template <typename In, bool FUSED, int PART>
__global__ __launch_bounds__(kPickThreads) void k_beam_pick(BeamArgs a) {
  __shared__ PickLds s;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int total = a.beams * a.parts, blocks = (total + kWaves - 1) / kWaves;
  const int b = FUSED ? blockIdx.x / blocks : blockIdx.x;
  const int64_t row0 = (int64_t)b * a.beams;
  BeamPart* parts = static_cast<BeamPart*>(a.workspace) + row0 * a.parts;
  if constexpr (FUSED) {
    const int place = blockIdx.x - b * blocks, id = place * kWaves + wave, k = id / a.parts;
    const bool on = id < total && !(a.finished && a.finished[row0 + k]);
    PartValues<In, PART> p;
    if (on)
      p.load(static_cast<const typename In::raw*>(a.logits) + (row0 + k) * a.row_stride, a.vocab,
             id - k * a.parts);
    exp64_table(s.table);  // while the logits come
    __syncthreads();
    BeamPart part;
    if (on) part = sum_part(p, s.table);
    if (blocks == 1) {
      if (on && lane == 0) s.parts[id] = part;
    } else {
      if (on && lane == 0) {
        uint64_t* w = reinterpret_cast<uint64_t*>(parts + id);
        store_agent(w, __builtin_bit_cast(uint64_t, part.sum));
        store_agent(w + 1, __float_as_uint(part.max));
      }
      stores_done();
      if (!last_of(a.marks + (int64_t)b * blocks, 1, blocks, place, a.tag, &s.count)) return;
      for (int i = threadIdx.x; i < total; i += kPickThreads) {
        const uint64_t* w = reinterpret_cast<const uint64_t*>(parts + i);
        const uint64_t sum = load_agent(w), max = load_agent(w + 1);
        s.parts[i] = BeamPart{__builtin_bit_cast(double, sum), __uint_as_float((uint32_t)max), 0};
      }
    }
    parts = s.parts;
  } else {
    exp64_table(s.table);
  }
  __syncthreads();

  for (int k = wave; k < a.beams; k += kWaves) {
    double lse = 0.0;
    if (!(a.finished && a.finished[row0 + k])) {
      const BeamPart* p = parts + (int64_t)k * a.parts;
      float m = -INFINITY;
      for (int i = lane; i < a.parts; i += 64) m = fmaxf(m, p[i].max);
      m = wave_all_max(m);
      const Exp64 ex(s.table, m);
      double sum = 0.0;
      for (int i = lane; i < a.parts; i += 64)
        if (p[i].max > -INFINITY) sum = __builtin_fma(p[i].sum, ex(p[i].max, 0.0), sum);
      sum = wave_all_sum(sum);
      lse = m < INFINITY ? (double)m + log(sum) : NAN;  // a row with +inf has no candidates
    }
    if (lane == 0) {
      s.lse[k] = lse;
      s.score[k] = a.scores[row0 + k];
    }
  }
  __syncthreads();

  // the n parts with the best maxima; a place is (beam, part) and then (beam, token)
  const int chunks = (a.parts + 63) / 64;
  auto each_part = [&](auto&& f) {
    for (int i = wave; i < a.beams * chunks; i += kWaves) {
      const int k = i / chunks, part = (i - k * chunks) * 64 + lane;
      if (part >= a.parts) continue;
      Cand c{-INFINITY, (int64_t)k << 32 | part};
      if (a.finished && a.finished[row0 + k]) {
        if (part == 0) c.score = s.score[k];
      } else {
        const float m = parts[k * a.parts + part].max;
        if (m > -INFINITY) c.score = s.score[k] + ((double)m - s.lse[k]);
      }
      if (c.score > -INFINITY) f(c);
    }
  };
  float top = -INFINITY;
  each_part([&](const Cand& c) { top = fmaxf(top, __double2float_rd(c.score)); });
  Cand bound{nth_of_tops(s, top, a.n), kNowhere - 1};
  const int picks = pick(s, a.n, bound, each_part);

  // the n best of their elements: no worse than the worst part's best
  for (int q = threadIdx.x; q < picks; q += kPickThreads) s.part[q] = s.chosen[q].at;
  bound.score = picks < a.n ? -INFINITY : s.chosen[picks - 1].score;
  __syncthreads();
  auto each_value = [&](auto&& f) {
#pragma unroll 1
    for (int q = wave; q < picks; q += kWaves) {
      const int k = (int)(s.part[q] >> 32), part = (int)s.part[q];
      const double sc = s.score[k], lse = s.lse[k];
      if (a.finished && a.finished[row0 + k]) {
        if (lane == 0) f(Cand{sc, (int64_t)k << 32 | a.eos_id});
        continue;
      }
      const typename In::raw* row =
          static_cast<const typename In::raw*>(a.logits) + (row0 + k) * a.row_stride;
      PartValues<In, PART> p;
      p.load(row, a.vocab, part);
      // what may pass, by a bound in 32 bits from below (less the roundings of 64 bits, of
      // which a score of -1e30 leaves nothing of the logit); those few are read once more
      const double slack = 1e-9 + 1e-15 * (fabs(bound.score) + fabs(sc) + fabs(lse));
      const float least = __double2float_rd(bound.score - sc + lse - slack);
      uint32_t good = 0;
#pragma unroll
      for (int i = 0; i < p.WORDS; ++i)
#pragma unroll
        for (int e = 0; e < In::N; ++e) good |= (uint32_t)(p.x[i][e] >= least) << (i * In::N + e);
      for (; good; good &= good - 1) {
        const int at = __builtin_ctz(good), v = p.token(at / In::N, at % In::N);
        const double score =
            v >= 0 && v < a.vocab ? sc + ((double)In::value(row[v]) - lse) : -INFINITY;
        if (score >= bound.score && score > -INFINITY) f(Cand{score, (int64_t)k << 32 | v});
      }
    }
  };
  // Where a beam has few parts, the n best reach into beams whose best is far behind the
  // best beam's values: a bound from the values then (10 requests of 13 beams, 900
  // tokens: 80 -> 16 us).
  if (picks < a.n || a.parts < 4 * a.n) {
    top = -INFINITY;
    for (int q = wave; q < picks; q += kWaves) {
      const int k = (int)(s.part[q] >> 32);
      double best = -INFINITY;
      if (a.finished && a.finished[row0 + k]) {
        if (lane == 0) best = s.score[k];
      } else {
        PartValues<In, PART> p;
        p.load(static_cast<const typename In::raw*>(a.logits) + (row0 + k) * a.row_stride, a.vocab,
               (int)s.part[q]);
        float x = -INFINITY;
#pragma unroll
        for (int i = 0; i < p.WORDS; ++i)
#pragma unroll
          for (int e = 0; e < In::N; ++e) x = fmaxf(x, p.x[i][e]);
        if (x > -INFINITY) best = s.score[k] + ((double)x - s.lse[k]);
      }
      top = fmaxf(top, __double2float_rd(best));
    }
    bound.score = fmax(bound.score, (double)nth_of_tops(s, top, a.n));
  }
  const int found = pick(s, a.n, bound, each_value);
  for (int r = threadIdx.x; r < a.n; r += kPickThreads) {
    const int64_t o = (int64_t)b * a.n + r;
    const bool any = r < found;
    const Cand c = any ? s.chosen[r] : kNone;
    const int k = any ? (int)(c.at >> 32) : -1, v = any ? (int)c.at : -1;
    a.out_scores[o] = any ? (float)c.score : -INFINITY;
    a.out_parents[o] = any ? (int)(row0 + k) : -1;
    a.out_tokens[o] = v;
    if (a.out_finished)
      a.out_finished[o] = any && ((a.finished && a.finished[row0 + k]) || v == a.eos_id);
  }
}

// rows that start off a 16-byte boundary have up to 7 values ahead of their first
int parts_of(int vocab, int part) { return (vocab + 7 + part - 1) / part; }

template <typename In, int PART>
hipError_t launch_one(BeamArgs a, hipStream_t st) {
  const int64_t total = (int64_t)a.beams * a.parts;
  a.tag = launch_tag();
  a.marks = reinterpret_cast<uint64_t*>(static_cast<BeamPart*>(a.workspace) + a.batch * total);
  k_beam_pick<In, true, PART>
      <<<(int)(a.batch * ((total + kWaves - 1) / kWaves)), kPickThreads, 0, st>>>(a);
  return hipGetLastError();
}

// One launch while all of its workgroups, of sixteen parts each, run at once (4 beams of
// 262144 tokens: 15 us, two launches 21), with small parts where there is room for them
// (large ones 17); more workgroups than that stream better as small ones of their own.
template <typename In>
hipError_t launch(BeamArgs a, hipStream_t st) {
  auto fits = [&](int parts) {
    const int64_t total = (int64_t)a.beams * parts;
    return total <= kFusedParts && a.batch * ((total + kWaves - 1) / kWaves) <= tune().cus;
  };
  a.parts = parts_of(a.vocab, kSmallPart);
  if (fits(a.parts)) return launch_one<In, kSmallPart>(a, st);
  a.parts = parts_of(a.vocab, kPart);
  if (fits(a.parts)) return launch_one<In, kPart>(a, st);
  const int64_t blocks = ((int64_t)a.batch * a.beams * a.parts + 3) / 4;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  k_beam_parts<In><<<(int)blocks, 256, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  k_beam_pick<In, false, kPart><<<a.batch, kPickThreads, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

// the parts, and a mark for each workgroup (there are no more of them than parts)
size_t beam_workspace(int64_t rows, int vocab) {
  return (size_t)rows * parts_of(vocab, kSmallPart) * (sizeof(BeamPart) + sizeof(uint64_t));
}

hipError_t launch_beam_select(const BeamArgs& a, int dtype_bytes, bool f16, hipStream_t st) {
  if (dtype_bytes == 4) return launch<F32In>(a, st);
  return f16 ? launch<F16In>(a, st) : launch<Bf16In>(a, st);
}

}  // namespace bq
