// Rotary positions of a step's queries and keys, with the per-head RMS norms
// where the model has them, and the writing of keys and values into the pages
// of the 16-bit cache.
//
// Reference: butterquant/head_prep.mojo:9-36 (the norm and rotation of a head,
// there ahead of the int8 rotation), kernels/attention_ops.mojo:45-51 (PagedKV).
//
// Per token at position p and pair i < rope_half: angle = p * inv_freq[i],
//   (a, b) -> mscale * (a cos - b sin, b cos + a sin)
// on the pairs (i, pair_stride + i), or (2i, 2i + 1) where pair_stride is 0;
// the rest of a head passes.  The angle is one product in 64 bits, as turns,
// and its whole turns are taken off there: at position 2^20 an angle in 32 bits
// is off by up to 2^-5 rad.  What is left, at most half a turn, goes to the
// sine and cosine instructions in 32 bits (2^-26 turns).
//
// Bound: every value is read once and written once (2159 tokens of 48 heads of 128: 14 us,
// 3.8 TB/s; a copy of that size moves 5.0); a decode step is one launch's latency (4.7 us).
#include "bq_half.hpp"
#include "bq_kernels.hpp"
#include "bq_pages.hpp"

namespace bq {

namespace {

constexpr int64_t kFullWaves = 2048;

// A wave takes 64 / LPH heads of one token at a time, head_dim / 8 = LPH lanes
// a head and 8 values a lane, IT times over, so that the sines of a lane's
// pairs serve IT heads and IT rows are on their way at once.
template <typename T, int LPH, int IT>
__global__ __launch_bounds__(256) void k_rope_append(RopeArgs a) {
  constexpr int HPW = 64 / LPH, HD = LPH * 8;
  const int heads = a.num_q + 2 * a.num_kv;
  const int groups = (heads + HPW * IT - 1) / (HPW * IT);
  const int64_t work = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t tok64 = work / groups;
  if (tok64 >= a.num_tokens) return;
  const int tok = __builtin_amdgcn_readfirstlane((int)tok64);
  const int group = __builtin_amdgcn_readfirstlane((int)(work - tok64 * groups));
  const int lane = lane_id(), c = lane % LPH, sub = lane / LPH;

  // this lane's pairs: values 8c .. 8c + 7 of a head, their partners in chunk pc
  int pc = c, i0 = 4 * c;
  float sign = 0.0f;  // of the partner's sine term; 0: these values pass
  if (a.pair_stride == 0) {
    sign = 8 * c < 2 * a.rope_half ? 1.0f : 0.0f;
  } else if (8 * c < a.rope_half) {
    i0 = 8 * c;
    pc = c + a.pair_stride / 8;
    sign = -1.0f;
  } else if (8 * c >= a.pair_stride && 8 * c < a.pair_stride + a.rope_half) {
    i0 = 8 * c - a.pair_stride;
    pc = c - a.pair_stride / 8;
    sign = 1.0f;
  }

  v4u x[IT], y[IT];
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int head = (group * IT + it) * HPW + sub;
    const bool is_q = head < a.num_q, is_k = head < a.num_q + a.num_kv;
    const uint16_t* src =
        is_q   ? a.q + (int64_t)tok * a.q_stride + (int64_t)head * HD
        : is_k ? a.k + (int64_t)tok * a.k_stride + (int64_t)(head - a.num_q) * HD
               : a.v + (int64_t)tok * a.v_stride + (int64_t)(head - a.num_q - a.num_kv) * HD;
    x[it] = y[it] = v4u{0, 0, 0, 0};
    if (head < heads) {
      x[it] = *reinterpret_cast<const v4u*>(src + 8 * c);
      if (pc != c && is_k) y[it] = *reinterpret_cast<const v4u*>(src + 8 * pc);
    }
  }

  const int pos = a.positions[tok];
  const int seq = a.seq_ids ? a.seq_ids[tok] : tok;
  if (pos < 0 || seq < 0 || seq >= a.num_seqs) return;  // padding
  const int64_t slot = page_slot(a.base_rows + (int64_t)seq * a.max_pages, a.max_pages,
                                 a.page_shift, a.num_slots, pos);
  float co[8], si[8];
  if (sign != 0.0f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (a.pair_stride == 0 && (e & 1)) {  // the pair of the value before
        co[e] = co[e - 1];
        si[e] = -si[e - 1];
        continue;
      }
      const int i = a.pair_stride == 0 ? i0 + e / 2 : i0 + e;
      const double turns = (double)pos * ((double)a.inv_freq[i] * 0.15915494309189533577);
      const float t = (float)(turns - __builtin_rint(turns));
      co[e] = a.mscale * __builtin_amdgcn_cosf(t);
      si[e] = a.mscale * __builtin_amdgcn_sinf(t) * (a.pair_stride == 0 ? -1.0f : sign);
    }
  }

#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int head = (group * IT + it) * HPW + sub;
    const bool is_q = head < a.num_q, is_k = !is_q && head < a.num_q + a.num_kv;
    const uint16_t* gain = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
    const bool norm = is_q || is_k ? gain != nullptr : a.norm_v != 0;
    const bool turn = sign != 0.0f && (is_q || is_k);
    float v[8], w[8];
    unpack8<T>(x[it], v);
    unpack8<T>(y[it], w);
    float ssq = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ssq = fmaf(v[e], v[e], ssq);
#pragma unroll
    for (int d = 1; d < LPH; d <<= 1) ssq += __shfl_xor(ssq, d);
    if (head >= heads || (!is_q && slot < 0)) continue;
    if (norm) {
      const float inv = a.sqrt_n / __builtin_sqrtf(ssq + a.n_eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= inv, w[e] *= inv;
      if (gain) {
        float g[8], gp[8];
        unpack8<T>(*reinterpret_cast<const v4u*>(gain + 8 * c), g);
        unpack8<T>(*reinterpret_cast<const v4u*>(gain + 8 * pc), gp);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= g[e], w[e] *= gp[e];
      }
    }
    v4u out = x[it];
    if (turn) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        o[e] = fmaf(a.pair_stride == 0 ? v[e ^ 1] : w[e], si[e], v[e] * co[e]);
      out = pack8<T>(o);
    } else if (norm) {
      out = pack8<T>(v);
    }
    uint16_t* dst =
        is_q ? a.q_out + (int64_t)tok * a.q_out_stride + (int64_t)head * HD
             : (is_k ? a.k_cache : a.v_cache) +
                   (slot * a.num_kv + (head - a.num_q - (is_k ? 0 : a.num_kv))) * (int64_t)HD;
    *reinterpret_cast<v4u*>(dst + 8 * c) = out;
  }
}

template <typename T, int LPH, int IT>
hipError_t launch_it(const RopeArgs& a, hipStream_t st) {
  const int per = 64 / LPH * IT, heads = a.num_q + 2 * a.num_kv;
  const int64_t blocks = ((int64_t)a.num_tokens * ((heads + per - 1) / per) + 3) / 4;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  k_rope_append<T, LPH, IT><<<(int)blocks, 256, 0, st>>>(a);
  return hipGetLastError();
}

// Four times the heads per wave once that still leaves kFullWaves waves (2159 tokens of 48
// heads: 16.8 -> 14.7 us).
template <typename T, int LPH>
hipError_t launch(const RopeArgs& a, hipStream_t st) {
  const int64_t lanes = (int64_t)a.num_tokens * (a.num_q + 2 * a.num_kv) * LPH;
  return lanes >= kFullWaves * 64 * 4 ? launch_it<T, LPH, 4>(a, st) : launch_it<T, LPH, 1>(a, st);
}

template <typename T>
hipError_t launch_hd(const RopeArgs& a, int head_dim, hipStream_t st) {
  switch (head_dim) {
    case 64: return launch<T, 8>(a, st);
    case 128: return launch<T, 16>(a, st);
    case 256: return launch<T, 32>(a, st);
    default: return launch<T, 64>(a, st);
  }
}

}  // namespace

hipError_t launch_rope_append(const RopeArgs& a, int head_dim, bool f16, hipStream_t st) {
  return f16 ? launch_hd<F16>(a, head_dim, st) : launch_hd<Bf16>(a, head_dim, st);
}

}  // namespace bq
