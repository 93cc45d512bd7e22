// Attention of one new token per sequence over the paged 16-bit cache.
//
// Reference: kernels/attention_ops.mojo:45-51 (PagedKV), :166-182 (online
// softmax of a tile), kernels/logsum_merge.mojo:29-122 (merge of the splits).
//
// Sequence s has one query row per head, at position len - 1, and attends to the
// cached positions [max(0, len - window), len):
//   x_p = cap tanh(scale q.k_p / cap),  o = sum_p e^(x_p) v_p / sum_p e^(x_p).
//
// Bound: the cache rows, 2 len num_kv head_dim 16-bit values per sequence, are
// read once; the arithmetic is 2 num_q / num_kv operations a byte.
//
// A wave walks tiles of TP positions for up to 16 query heads of one kv head.
// Scores: A = 16 cache rows, B = the 16 query heads (those past the group are
// zero), so a lane ends with 4 positions of one head per 16 rows.  That is the
// layout in which the next product takes its B operand when a tile's positions
// are read as its k index in the order (group of 16, quad, row): the weights go
// from one product to the next in their lane.  The values are the other operand,
// transposed, as O^T = V^T P^T: a lane reads 8 columns of its positions (16 lanes:
// 256 contiguous bytes of a row) and pairs positions with one byte permute per
// two values.  No LDS and no cross-lane traffic but the maxima.
// Weights go to that product as two values of the cache's type, the second what
// rounding the first leaves (2^-16 or 2^-22 of the weight are lost; one value alone
// would cost as much again as the output's own rounding, and saves 1% of the time);
// scores, maxima, sums and outputs are 32 bits until the one rounding at the end.
//
// The waves of a workgroup take every NW-th tile of a range and join in LDS; the ranges
// of a sequence are joined in their order, by the last of its workgroups or, where that
// is much, by k_paged_merge.
//
// 64 sequences of 14 to 16 thousand positions, 8 kv heads of 128: 697 us, 5.7 TB/s (a
// large read reaches 6.0); 16 of 4096, 2 kv heads of 512: 49 + 5 us, 4.7 TB/s.
#include <algorithm>

#include "bq_half.hpp"
#include "bq_kernels.hpp"
#include "bq_pages.hpp"

namespace bq {

namespace {

constexpr float kLn2 = 0.6931471805599453f;

__device__ inline float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// over the four lanes l % 16 + {0, 16, 32, 48}
__device__ inline float quad_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ inline float quad_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Partial sums that the attention's last workgroup joins itself, instead of a launch of
// k_paged_merge (1 x 1024 positions: 13.8 -> 11.2 us; 16 x 8000 positions of one kv head
// with 131 KB of them: 22.8 -> 29.7).
constexpr int64_t kJoinBytes = 48 << 10;  // of a sequence of mean length; twice that at most
constexpr int kJoinMost = 128;            // splits
constexpr int kMlStride = 4;  // floats of workspace per split beside its sums: m, l, mark
// where there are no marks: a sequence's first slot and its splits, for k_paged_merge
__device__ inline int2* plan_of(const PagedAttnArgs& a, int seq) {
  return reinterpret_cast<int2*>(a.ws_ml + (int64_t)seq * kMlStride + 2);
}

// Parts of one row joined: sums scaled from each part's maximum to the common one.
template <typename T>
struct Joined {
  float ms, M, L = 0.0f;
  v4f32 acc = {0, 0, 0, 0};
  __device__ void start(float max) {
    M = max;
    ms = max == -INFINITY ? 0.0f : max;
  }
  __device__ void add(float m, float l, v4f32 v) {
    const float f = exp2_(m - ms);
    L = fmaf(f, l, L);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(f, v[i], acc[i]);
  }
  __device__ void store(const PagedAttnArgs& a, int64_t row, int hd, int col) const {
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;  // a NaN sum stays
    const v2u w = {T::pack(acc[0] * inv, acc[1] * inv), T::pack(acc[2] * inv, acc[3] * inv)};
    *reinterpret_cast<v2u*>(a.out + row * hd + col) = w;
    if (a.lse && col == 0)
      a.lse[row] = L != 0.0f ? (M + __builtin_amdgcn_logf(L) - T::kWeightBits) * kLn2 : -INFINITY;
  }
};

// a sequence's positions [start, len) and its tiles [first, end) of TP positions
struct Span {
  int len, start, first, end;
};

__device__ inline Span attn_span(const PagedAttnArgs& a, int kv_len, int tp) {
  Span r;
  const int64_t room = (int64_t)a.max_pages << a.page_shift;
  const int64_t len = kv_len < room ? kv_len : room;
  r.len = (int)(len > 0 ? len : 0);
  r.start = a.window > 0 && r.len > a.window ? r.len - a.window : 0;
  r.first = r.start / tp, r.end = (int)(((int64_t)r.len + tp - 1) / tp);
  return r;
}

// What a workgroup takes: split `split` of the `splits` of sequence `seq` (-1: nothing),
// whose partial sums begin at `slot0`.
struct Work {
  int seq, split, splits, slot0;
  int kv_len;  // the sequence's entry
};

// Shares the slots out by length (attn_splits): 64 sequences, one of 65536 positions and
// 63 of 512, 8 kv heads of 128: 815 us with one workgroup each, 89 shared out.  Every wave
// works it out from the lengths, a lane for every 64th part of the sequences.  From two
// units a sequence on, the longest split counts: the largest share that rounded up fills
// no more than `units` (64 of 1 to 8192 positions, 4 kv heads of 256, 2 units each: 276
// rounded down, 223).  Taking the longest first would help where long ones meet on a
// compute unit, but every wave's sort costs as much (64 of 300: 17.6 -> 24.5 us).
__device__ inline Work attn_work(const PagedAttnArgs& a, int slot, int tp) {
  if (a.s_max == 1) return {slot, 0, 1, 0, a.kv_lens[slot]};
  auto tiles = [&](int kv_len) {
    const Span r = attn_span(a, kv_len, tp);
    return r.end - r.first;
  };
  if (a.num_seqs == 1) {
    const int t = tiles(a.kv_lens[0]);
    const int n = attn_splits(t, t > 0 ? (double)a.units / t : 0.0, kRoundDown, a.n_max);
    return {slot < n ? 0 : -1, slot, n, 0, a.kv_lens[0]};
  }
  const int lane = lane_id(), per = (a.num_seqs + 63) / 64;
  const int s0 = min(lane * per, a.num_seqs), s1 = min(s0 + per, a.num_seqs);
  Work w{s0, 0, 1, 0, 0};
  auto sum = [](auto x) { return wave_all(x, [](auto p, auto q) { return p + q; }); };
  const bool up = attn_rounds_up(a.num_seqs, a.units);
  const double round = up ? kRoundUp : kRoundDown;
  double share;
  int mine = 0;
  if (per == 1) {
    const bool on = s0 < s1;
    w.kv_len = on ? a.kv_lens[s0] : 0;
    const int t = tiles(w.kv_len);
    auto count = [&](double x) { return on ? attn_splits(t, x, round, a.n_max) : 0; };
    const double all = sum((double)t);
    share = all > 0.0 ? a.units / all : 0.0;
    if (up && all > 0.0 && sum(count(share)) > a.units) {
      double lo = (a.units - a.num_seqs) / all, hi = share;
      for (int i = 0; i < 5; ++i) {
        const double mid = 0.5 * (lo + hi);
        (sum(count(mid)) <= a.units ? lo : hi) = mid;
      }
      share = lo;
    }
    w.splits = mine = count(share);
  } else {
    double all = 0.0;
    for (int s = s0; s < s1; ++s) all += tiles(a.kv_lens[s]);
    all = sum(all);
    share = all > 0.0 ? a.units / all : 0.0;
    for (int s = s0; s < s1; ++s) mine += attn_splits(tiles(a.kv_lens[s]), share, round, a.n_max);
  }
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int x = __shfl_up(upto, d);
    if (lane >= d) upto += x;
  }
  const uint64_t past = __ballot(upto > slot);
  if (past == 0) return {-1, 0, 1, 0, 0};
  const int from = __builtin_ctzll(past);
  w.slot0 = upto - mine;
  if (per > 1 && lane == from) {
    for (; w.seq < s1; ++w.seq) {
      w.kv_len = a.kv_lens[w.seq];
      w.splits = attn_splits(tiles(w.kv_len), share, round, a.n_max);
      if (w.slot0 + w.splits > slot) break;
      w.slot0 += w.splits;
    }
    if (w.seq == s1) w.seq = -1;  // lengths that changed meanwhile
  }
  w.seq = __builtin_amdgcn_readlane(w.seq, from);
  w.splits = __builtin_amdgcn_readlane(w.splits, from);
  w.slot0 = __builtin_amdgcn_readlane(w.slot0, from);
  w.kv_len = __builtin_amdgcn_readlane(w.kv_len, from);
  w.split = slot - w.slot0;
  return w;
}

// From HD = 256 on, 16 positions a tile: K, V, the queries and the accumulators of 32
// would pass the registers that leave room for two waves (HD = 512: for one).
template <int HD>
constexpr int tile_positions() {
  return HD >= 256 ? 16 : 32;
}

// HD = 256 keeps its queries in LDS, which makes room for three waves (8 sequences of
// 8000 positions, 8 kv heads: 125 -> 93 us); HD = 512 has one wave either way, which
// would wait for them (16 x 4096 positions, 2 kv heads: 52 -> 60 us).
template <int HD>
constexpr bool queries_in_lds() {
  return HD == 256;
}

// Pages of fewer than 16 rows (SMALL) are looked up position by position and their
// slots passed between lanes; larger ones once per 16 positions, with the wave's
// address in scalar registers and the lanes' offsets the same for every tile.
//
// The next tile's rows are asked for as soon as the registers of this one's are free:
// K behind the scores, V behind the value product.
template <typename T, int HD, int NW, bool SMALL>
__global__ __launch_bounds__(NW * 64, HD == 512 ? 1 : 3) void k_paged_attn(
    PagedAttnArgs a) {
  constexpr int TP = tile_positions<HD>();
  constexpr int KS = HD / 32;            // steps of the score product
  constexpr int MT = TP / 16;            // groups of 16 positions
  constexpr int CPL = HD == 64 ? 4 : 8;  // value columns per lane and group
  constexpr int CG = HD / (16 * CPL);    // column groups
  constexpr int VW = CPL / 2;            // words of a value load
  constexpr int NP = TP / 4;             // positions per lane of the value product
  constexpr int LD = HD + 8;             // LDS row: 16 heads 32 bytes apart in the banks
  constexpr uint32_t FULL = (uint32_t)((1ull << TP) - 1);
  constexpr bool QLDS = queries_in_lds<HD>();

  extern __shared__ float smem[];  // QLDS: queries; acc [NW][G][LD], m, l [NW][16] each; a flag
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, quad = lane >> 4;

  // Workgroups go to the 8 dies in turn: those on the same rows (the groups of 16 query
  // heads of a kv head) are 8 apart, on one die and its cache.
  int b = blockIdx.x, hg = 0;
  if (a.head_groups > 1) {
    hg = b / 8 % a.head_groups;
    b = b / (8 * a.head_groups) * 8 + b % 8;
    if (b >= a.num_seqs * a.num_kv * a.s_max) return;
  }
  const int kvh = b % a.num_kv;
  const Work wk = attn_work(a, b / a.num_kv, TP);
  if (wk.seq < 0) return;
  const int seq = wk.seq;
  const int G = min(16, a.gqa - hg * 16);
  const int head0 = kvh * a.gqa + hg * 16;

  const Span rg = attn_span(a, wk.kv_len, TP);
  const int each = (rg.end - rg.first) / wk.splits, odd = (rg.end - rg.first) % wk.splits;
  const int t0 = rg.first + wk.split * each + min(wk.split, odd);
  const int t1 = t0 + each + (wk.split < odd ? 1 : 0);

  // the queries: in registers, or (large heads) in LDS for all waves
  v4u qf[KS];
  v4u* qs = reinterpret_cast<v4u*>(smem);  // [KS][64]
  float* part = smem + (QLDS ? KS * 256 : 0);
  {
    const uint16_t* q = a.q + (int64_t)seq * a.q_stride + (int64_t)(head0 + n16) * HD + quad * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      if (!QLDS || ks % NW == wave)
        qf[ks] = n16 < G ? *reinterpret_cast<const v4u*>(q + ks * 32) : v4u{0, 0, 0, 0};
  }

  const int32_t* rows = a.base_rows + (int64_t)seq * a.max_pages;
  const int64_t stride = (int64_t)a.num_kv * HD;
  const uint16_t* kc = a.k_cache + (int64_t)kvh * HD;
  const uint16_t* vc = a.v_cache + (int64_t)kvh * HD;
  const uint32_t koff = (uint32_t)(n16 * stride + quad * 8) * 2;
  uint32_t voff[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) voff[r] = (uint32_t)((quad * 4 + r) * stride + n16 * CPL) * 2;

  // a tile's rows: its slots (SMALL: of position lane % TP; else of the first row of each
  // 16, the same in all lanes) and which of its positions take part
  struct Tile {
    uint32_t ok;
    int32_t slot[SMALL ? 1 : MT];
  };
  auto find = [&](int t) {
    Tile x;
    const int p0 = t * TP;
    if constexpr (SMALL) {
      const int p = p0 + (lane & (TP - 1));
      const bool in = p >= rg.start && p < rg.len;
      const int64_t s = in ? page_slot(rows, a.max_pages, a.page_shift, a.num_slots, p) : -1;
      x.ok = (uint32_t)__ballot(s >= 0) & FULL;
      x.slot[0] = s < 0 ? 0 : (int)s;
    } else {
      x.ok = FULL;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int p = p0 + i * 16;
        // past the end there may be no entry: nothing of these 16 takes part
        const int32_t base = p < rg.len ? rows[p >> a.page_shift] : -1;
        const bool in = page_in(base, a.page_shift, a.num_slots);
        x.slot[i] = in ? base + (p & ((1 << a.page_shift) - 1)) : 0;
        if (!in) x.ok &= ~(0xFFFFu << (16 * i));
      }
      if (p0 + TP > rg.len) x.ok &= (uint32_t)((1ull << (rg.len - p0)) - 1);
      if (p0 < rg.start) x.ok &= ~(uint32_t)((1ull << (rg.start - p0)) - 1);
    }
    return x;
  };
  v4u kf[MT][KS];
  uint32_t vf[CG][NP][VW];
  auto load_k = [&](const Tile& x) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const char* p;
      if constexpr (SMALL)
        p = reinterpret_cast<const char*>(kc + __shfl(x.slot[0], i * 16 + n16) * stride +
                                          quad * 8);
      else
        p = reinterpret_cast<const char*>(kc + x.slot[i] * stride) + koff;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[i][ks] = *reinterpret_cast<const v4u*>(p + ks * 64);
    }
  };
  auto load_v = [&](const Tile& x) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const char* p;
      if constexpr (SMALL)
        p = reinterpret_cast<const char*>(
            vc + __shfl(x.slot[0], (j >> 2) * 16 + quad * 4 + (j & 3)) * stride + n16 * CPL);
      else
        p = reinterpret_cast<const char*>(vc + x.slot[j >> 2] * stride) + voff[j & 3];
#pragma unroll
      for (int i = 0; i < CG; ++i) {
        if constexpr (VW == 4) {
          const v4u w = *reinterpret_cast<const v4u*>(p + i * 256);
#pragma unroll
          for (int x = 0; x < 4; ++x) vf[i][j][x] = w[x];
        } else {
          const v2u w = *reinterpret_cast<const v2u*>(p);
          vf[i][j][0] = w[0];
          vf[i][j][1] = w[1];
        }
      }
    }
  };

  v4f32 o[CG][CPL];
#pragma unroll
  for (int i = 0; i < CG; ++i)
#pragma unroll
    for (int c = 0; c < CPL; ++c) o[i][c] = v4f32{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;

  int t = t0 + wave;
  Tile cur{}, next{};
  if (t < t1) {
    cur = find(t);
    load_k(cur);
    load_v(cur);
    if (t + NW < t1) next = find(t + NW);
  }
  if constexpr (QLDS) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      if (ks % NW == wave) qs[ks * 64 + lane] = qf[ks];
    __syncthreads();
  }
  for (; t < t1; t += NW) {
    const bool more = t + NW < t1;
    // scores in powers of two, -inf where a position takes no part
    float x[NP];
    float mt = -INFINITY;
    v4f32 sc[MT];
    int here = lane;
    if constexpr (QLDS) asm volatile("" : "+v"(here));  // read again, not kept in registers
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      sc[i] = v4f32{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sc[i] = T::mfma32(kf[i][ks], QLDS ? qs[ks * 64 + here] : qf[ks], sc[i]);
    }
    if (more) load_k(next);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float y = sc[i][r] * a.scale2;
        if (a.softcap2 > 0.0f) {  // cap tanh(y / cap), tanh z = 1 - 2 / (e^2z + 1)
          const float e = exp2_(y * a.inv_cap);
          y = a.softcap2 * (1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f));
        }
        y = (cur.ok >> (i * 16 + quad * 4 + r)) & 1 ? y : -INFINITY;
        x[i * 4 + r] = y;
        mt = fmaxf(mt, y);
      }
    }
    const float mn = fmaxf(m, quad_max(mt));
    const float ms = mn == -INFINITY ? 0.0f : mn;
    const float alpha = exp2_(m - ms), mw = ms - T::kWeightBits;
    m = mn;
    uint32_t pf[NP / 2], pl[NP / 2];  // the weights, and what rounding them leaves
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NP; j += 2) {
      const float p0_ = exp2_(x[j] - mw), p1_ = exp2_(x[j + 1] - mw);
      sum += p0_ + p1_;
      pf[j / 2] = T::pack(p0_, p1_);
      pl[j / 2] = T::pack(p0_ - T::lo(pf[j / 2]), p1_ - T::hi(pf[j / 2]));
    }
    l = fmaf(l, alpha, sum);
    if (cur.ok != FULL) {  // what stands in other rows may be anything
#pragma unroll
      for (int j = 0; j < NP; ++j)
        if (!((cur.ok >> ((j >> 2) * 16 + quad * 4 + (j & 3))) & 1))
#pragma unroll
          for (int i = 0; i < CG; ++i)
#pragma unroll
            for (int w = 0; w < VW; ++w) vf[i][j][w] = 0;
    }
#pragma unroll
    for (int i = 0; i < CG; ++i)
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const uint32_t sel = c & 1 ? 0x07060302u : 0x05040100u;
        uint32_t vt[NP / 2];
#pragma unroll
        for (int j = 0; j < NP / 2; ++j)
          vt[j] = __builtin_amdgcn_perm(vf[i][2 * j + 1][c / 2], vf[i][2 * j][c / 2], sel);
        v4f32 acc = o[i][c] * alpha;
        if constexpr (NP == 8) {
          const v4u v = {vt[0], vt[1], vt[2], vt[3]};
          acc = T::mfma32(v, v4u{pf[0], pf[1], pf[2], pf[3]}, acc);
          acc = T::mfma32(v, v4u{pl[0], pl[1], pl[2], pl[3]}, acc);
        } else {
          const v2u v = {vt[0], vt[1]};
          acc = T::mfma16(v, v2u{pf[0], pf[1]}, acc);
          acc = T::mfma16(v, v2u{pl[0], pl[1]}, acc);
        }
        o[i][c] = acc;
      }
    if (more) load_v(next);
    cur = next;
    if (t + 2 * NW < t1) next = find(t + 2 * NW);
  }
  l = quad_sum(l);

  // the waves' parts, joined in LDS: o[i][c][r] is column i 16 CPL + (4 quad + r) CPL + c
  float* sm = part + (size_t)NW * G * LD;
  if (n16 < G) {
    float* d = part + ((size_t)wave * G + n16) * LD;
#pragma unroll
    for (int i = 0; i < CG; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < CPL; c += 4)
          *reinterpret_cast<v4f32*>(d + i * 16 * CPL + (quad * 4 + r) * CPL + c) =
              v4f32{o[i][c][r], o[i][c + 1][r], o[i][c + 2][r], o[i][c + 3][r]};
    if (quad == 0) {
      sm[wave * 16 + n16] = m;
      sm[NW * 16 + wave * 16 + n16] = l;
    }
  }
  __syncthreads();
  const int64_t row0 = (int64_t)seq * a.num_q + head0;
  const bool whole = wk.splits <= 1;
  const int64_t slots = (int64_t)a.num_seqs * a.s_max;
  for (int e = threadIdx.x; e < G * (HD / 4); e += NW * 64) {
    const int h = e / (HD / 4), col = (e % (HD / 4)) * 4;
    Joined<T> j;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w * 16 + h]);
    j.start(M);
#pragma unroll
    for (int w = 0; w < NW; ++w)
      j.add(sm[w * 16 + h], sm[NW * 16 + w * 16 + h],
            *reinterpret_cast<const v4f32*>(part + ((size_t)w * G + h) * LD + col));
    if (whole) {
      j.store(a, row0 + h, HD, col);
    } else {
      const int64_t at = (head0 + h) * slots + wk.slot0 + wk.split;
      store_agent(a.ws_acc + at * HD + col, j.acc[0], j.acc[1]);
      store_agent(a.ws_acc + at * HD + col + 2, j.acc[2], j.acc[3]);
      if (col == 0) store_agent(a.ws_ml + at * kMlStride, M, j.L);
    }
  }
  if (!a.tag && a.s_max > 1 && kvh == 0 && hg == 0 && wk.split == 0 && threadIdx.x == 0)
    *plan_of(a, seq) = int2{wk.slot0, wk.splits};
  if (whole || !a.tag) return;

  // the splits are joined by whoever comes last
  stores_done();
  uint64_t* marks = reinterpret_cast<uint64_t*>(a.ws_ml + (head0 * slots + wk.slot0) * kMlStride + 2);
  if (!last_of(marks, kMlStride / 2, wk.splits, wk.split, a.tag,
               reinterpret_cast<int*>(sm + 2 * NW * 16)))
    return;
  // Maxima and sums to LDS, over the waves' parts; then eight splits' sums at a time.
  static_assert(2 * kJoinMost <= NW * LD, "room for the splits' m and l of each head");
  for (int e = threadIdx.x; e < G * wk.splits; e += NW * 64) {
    const int h = e / wk.splits, i = e - h * wk.splits;
    const v2f v = load2_agent(a.ws_ml + ((head0 + h) * slots + wk.slot0 + i) * kMlStride);
    part[2 * e] = v[0];
    part[2 * e + 1] = v[1];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < G * (HD / 4); e += NW * 64) {
    const int h = e / (HD / 4), col = (e % (HD / 4)) * 4;
    const float* ml = part + 2 * h * wk.splits;
    const float* acc = a.ws_acc + ((head0 + h) * slots + wk.slot0) * HD + col;
    Joined<T> j;
    float M = -INFINITY;
    for (int i = 0; i < wk.splits; ++i) M = fmaxf(M, ml[2 * i]);
    j.start(M);
    for (int i0 = 0; i0 < wk.splits; i0 += 8) {
      v2f lo[8], hi[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < wk.splits) {
          lo[i] = load2_agent(acc + (int64_t)(i0 + i) * HD);
          hi[i] = load2_agent(acc + (int64_t)(i0 + i) * HD + 2);
        }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < wk.splits)
          j.add(ml[2 * (i0 + i)], ml[2 * (i0 + i) + 1], v4f32{lo[i][0], lo[i][1], hi[i][0], hi[i][1]});
    }
    j.store(a, row0 + h, HD, col);
  }
}

// Joins a row's splits in their order: HD / 4 lanes a row, four columns each.
template <typename T, int HD>
__global__ __launch_bounds__(256) void k_paged_merge(PagedAttnArgs a) {
  constexpr int TPR = HD / 4, RPB = 256 / TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (row >= (int64_t)a.num_seqs * a.num_q) return;
  const int seq = (int)(row / a.num_q), col = (threadIdx.x % TPR) * 4;
  const int2 plan = *plan_of(a, seq);
  const int S = plan.y;
  if (S <= 1) return;
  const int64_t at = row % a.num_q * ((int64_t)a.num_seqs * a.s_max) + plan.x;
  const float* ml = a.ws_ml + at * kMlStride;
  const float* acc = a.ws_acc + at * HD + col;
  Joined<T> j;
  float M = -INFINITY;
  for (int s = 0; s < S; ++s) M = fmaxf(M, ml[s * kMlStride]);
  j.start(M);
#pragma unroll 4
  for (int s = 0; s < S; ++s)
    j.add(ml[s * kMlStride], ml[s * kMlStride + 1],
          *reinterpret_cast<const v4f32*>(acc + (int64_t)s * HD));
  j.store(a, row, HD, col);
}

template <typename T, int HD, bool SMALL>
hipError_t launch_attn(const PagedAttnArgs& a, hipStream_t st) {
  constexpr int NW = 4;
  const int G = std::min(16, a.gqa);
  const bool up = attn_rounds_up(a.num_seqs, a.units);  // fills no more than the units
  int64_t blocks = (up ? a.units : (int64_t)a.num_seqs * a.s_max) * a.num_kv;
  if (a.head_groups > 1) blocks = (blocks + 7) / 8 * 8 * a.head_groups;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  const size_t lds = ((size_t)NW * G * (HD + 8) + 2 * NW * 16 + 4 + (queries_in_lds<HD>() ? HD * 8 : 0)) *
                     sizeof(float);
  if (lds > 65536) {
    const hipError_t e =
        hipFuncSetAttribute(reinterpret_cast<const void*>(&k_paged_attn<T, HD, NW, SMALL>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  k_paged_attn<T, HD, NW, SMALL><<<(int)blocks, NW * 64, lds, st>>>(a);
  return hipGetLastError();
}

template <typename T, int HD>
hipError_t launch(PagedAttnArgs a, hipStream_t st) {
  const int64_t row_bytes = (int64_t)std::min(16, a.gqa) * HD * 4;  // of a split's sums
  a.units = attn_units(a.num_seqs, a.s_max);
  const bool fused = a.s_max > 1 && a.units / a.num_seqs * row_bytes <= kJoinBytes;
  a.n_max = fused ? (int)std::min<int64_t>(kJoinMost, 2 * kJoinBytes / row_bytes) : 256;
  a.tag = fused ? launch_tag() : 0;
  const hipError_t e =
      a.page_shift < 4 ? launch_attn<T, HD, true>(a, st) : launch_attn<T, HD, false>(a, st);
  if (e != hipSuccess || a.s_max == 1 || fused) return e;
  const int rpb = 256 / (HD / 4);
  const int64_t rows = (int64_t)a.num_seqs * a.num_q;
  if ((rows + rpb - 1) / rpb > INT32_MAX) return hipErrorInvalidValue;
  k_paged_merge<T, HD><<<(int)((rows + rpb - 1) / rpb), 256, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_hd(const PagedAttnArgs& a, int hd, hipStream_t st) {
  switch (hd) {
    case 64: return launch<T, 64>(a, st);
    case 128: return launch<T, 128>(a, st);
    case 256: return launch<T, 256>(a, st);
    default: return launch<T, 512>(a, st);
  }
}

}  // namespace

// A workgroup (4 waves, a tile each at a time) per compute unit reads at the full rate
// and leaves the fewest sums to join: 8 sequences of 16384 positions, 8 kv heads of 128:
// 4 splits 104 us, 12 splits 105, 2 splits 137; 16 of 8000 with 32 query heads on one
// kv head: 8 splits 20, 24 splits 26.  Rounds of them should leave few units idle (8 kv
// heads of 128, 500 to 8000 positions: 12 sequences, 2 workgroups for each 38 us, 3 46; 20
// sequences: 1 110, 2 95, 3 81).  Where there are enough without splits, one for each, on
// average, evens out lengths; heads of 256 take two (64 of up to 8192, 4 kv heads: 257 us,
// two 223, equal lengths 349 and 364; heads of 128, 32 of up to 4096: 50 and 49, equal
// lengths 96 and 103).  Short ones do not need it (256 of 1000, one kv head of 128: 24,
// shared out 27).  A sequence of three rounds has one split (7 of 333 positions: 6.7, 3
// splits 7.2 us).
int paged_attn_splits(int num_seqs, int num_q, int num_kv, int head_dim, int max_kv_len, int window) {
  const int tp = head_dim >= 256 ? 16 : 32;
  const int64_t len = window > 0 ? std::min(max_kv_len, window) : max_kv_len;
  const int64_t tiles = (len + tp - 1) / tp + (window > 0 ? 1 : 0);
  const int64_t groups = (int64_t)num_seqs * num_kv * ((num_q / num_kv + 15) / 16);
  const int64_t cus = tune().cus;
  if (tiles <= 12) return 1;
  int64_t s;
  if (groups >= cus) {
    if (num_seqs == 1 || num_seqs > 1024 || tiles <= 48) return 1;
    s = head_dim == 256 ? 2 : 1;
  } else {
    s = cus / groups;
    while (10 * s * groups < 7 * cus * ((s * groups + cus - 1) / cus)) ++s;
  }
  return (int)std::min<int64_t>({s, (tiles + 5) / 6, 255}) + (num_seqs > 1);
}

hipError_t launch_paged_attn(const PagedAttnArgs& a, int head_dim, bool f16, hipStream_t st) {
  return f16 ? launch_hd<F16>(a, head_dim, st) : launch_hd<Bf16>(a, head_dim, st);
}

}  // namespace bq
