// The K/V cache in 4 or 8 bits: rows quantised as they are written, read back
// as bf16, and attended in their packed form.
//
// A row of one head (D = 64, 128 or 256 values) has D / 64 groups of 64
// values. A group stands for low + step * code, codes 0 .. T = 2^bits - 1:
//   low  = its least value (a bf16 value, so stored exactly),
//   step = bf16((greatest - low) / T), each operation rounded to fp32,
//   code = the whole number nearest to (x - low) / step, ties to even, in the
//          real numbers (no rounding decides it), held to 0 .. T;
// a group without a range has step 0 and codes 0; a group that holds a NaN or
// an infinity has step = low = NaN and reads back as NaN.
//
// Keys: group g is dims 64 g .. 64 g + 63. Values: group g is the dims d with
// (d mod D/16) div 4 == g, four neighbours of each of the row's 16 runs of D/16
// dims. The attention's P V product has lane c of 16 read run c of a token and
// feed the matrix cores one dim of every run at a time, so with these groups
// each such product has one scale per token.
//
// Layouts: codes [B, KVH, C, D * bits / 8] bytes, dims in order, in 4 bits the
// even dim in a byte's low half; params [B, KVH, D / 64, C] pairs of bf16
// (step in the low half of a 32-bit word, low in the high half).
#include "q35_common.hpp"

namespace {

Q35_DEV uint32_t kvq_code(uint32_t w, int i, int bits) { return bits == 4 ? (w >> (4 * i)) & 15u : (w >> (8 * i)) & 255u; }

// Whether a code's place between its neighbours has to be looked at exactly:
// t = (x - low) / step less the code, as computed with a reciprocal (relative
// error below 2^-21, so below 2^-13 for 255 steps).
Q35_DEV bool kvq_near(float t) { return !(fabsf(t) < 0.4995f); }

// The exact code of xh = x / 2 in a group with lh = low / 2 and sh = step / 2:
// halves, as x - low may pass the fp32 range; halving and (code +- 1/2) * sh
// (at most 17 bits) are exact, and so is the error e of s = xh - lh, so the
// borders are compared in the real numbers.
Q35_DEV float kvq_exact_code(float xh, float lh, float sh) {
  const float s = xh - lh;
  const float bb = s - xh;
  const float e = (xh - (s - bb)) + (-lh - bb);
  float c = rintf(s / sh);
  const bool odd = ((int)c & 1) != 0;
  const float hi = (c + 0.5f) * sh, lo = (c - 0.5f) * sh;
  if (s > hi || (s == hi && (e > 0.f || (e == 0.f && odd)))) c += 1.f;
  else if (s < lo || (s == lo && (e < 0.f || (e == 0.f && odd)))) c -= 1.f;
  return c;
}

// One group's step and low as the stored word, and its halves and reciprocal.
struct KvqGroup {
  uint32_t word;
  float lh, sh, inv;  // low / 2, step / 2, 2 / step (0 for step 0)
  bool exact;         // step too small for the reciprocal's error bound
};
template <int BITS>
Q35_DEV KvqGroup kvq_group(float lo, float hi) {
  constexpr float T = BITS == 4 ? 15.f : 255.f;
  KvqGroup g;
  const bool finite = lo > -INFINITY && hi < INFINITY;
  const float r = hi * 0.5f - lo * 0.5f;
  const uint32_t step = finite ? f2bf(r / (T * 0.5f)) : 0x7fc0u;
  g.word = step | (finite ? __float_as_uint(lo) & 0xffff0000u : 0x7fc00000u);
  g.lh = finite ? lo * 0.5f : 0.f;
  g.sh = finite ? bf2f(step) * 0.5f : 0.f;
  g.exact = g.sh < 1.0e-30f;
  g.inv = g.exact ? 0.f : 1.0f / g.sh;
  return g;
}
template <int BITS>
Q35_DEV uint32_t kvq_encode(float x, const KvqGroup& g) {
  constexpr float T = BITS == 4 ? 15.f : 255.f;
  const float q = fmaf(x, 0.5f, -g.lh) * g.inv;
  float c = rintf(q);
  if (kvq_near(q - c) || g.exact) c = g.sh > 0.f ? kvq_exact_code(x * 0.5f, g.lh, g.sh) : 0.f;
  return (uint32_t)fminf(fmaxf(c, 0.f), T);
}

// ------------------------------------------------------------------- write
// 16 lanes a row: lane c holds run c, dims E c .. E c + E - 1 (E = D / 16). A
// key group is 64 / E lanes wide, a value group 4 dims of all 16 lanes. Both
// grids (blockIdx.y: 0 keys, 1 values) read 2 D bytes and write D * bits / 8 +
// 4 D / 64 a row.
struct KvqSrc {
  const uint16_t* p;
  long long sb, sh, sl;  // strides of batch, head, token in elements
};
template <int E, int BITS>
__global__ __launch_bounds__(256) void kvq_write(const KvqSrc ks, const KvqSrc vs, uint8_t* __restrict__ kq,
                                                 uint8_t* __restrict__ vq, uint32_t* __restrict__ kp,
                                                 uint32_t* __restrict__ vp, const long long* start_dev,
                                                 int n_start, long long start, int KVH, int L, int C,
                                                 unsigned rows) {
  constexpr int NG = E / 4, RB = 2 * E * BITS;  // groups, bytes of a packed row
  const unsigned row = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (row >= rows) return;
  const int c = threadIdx.x & 15;
  const unsigned bh = row / (unsigned)L, t = row % (unsigned)L;
  const unsigned b = bh / (unsigned)KVH, h = bh % (unsigned)KVH;
  const long long pos = (start_dev ? start_dev[n_start > 1 ? b : 0] : 0) + start + t;
  const bool values = blockIdx.y != 0;
  const KvqSrc& s = values ? vs : ks;
  const uint16_t* src = s.p + (long long)b * s.sb + (long long)h * s.sh + (long long)t * s.sl + E * c;
  uint32_t w[E / 2];
  if constexpr (E == 4) {
    const uint2 a = *reinterpret_cast<const uint2*>(src);
    w[0] = a.x; w[1] = a.y;
  } else {
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      const uint4 a = *reinterpret_cast<const uint4*>(src + 8 * j);
      w[4 * j] = a.x; w[4 * j + 1] = a.y; w[4 * j + 2] = a.z; w[4 * j + 3] = a.w;
    }
  }
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = e & 1 ? bf_hi(w[e / 2]) : bf_lo(w[e / 2]);
  // Least and greatest value of 4 dims; a NaN (which min and max pass over)
  // shows as an infinite greatest value.
  float lo[NG], hi[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float* y = x + 4 * g;
    lo[g] = fminf(fminf(y[0], y[1]), fminf(y[2], y[3]));
    hi[g] = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
    const float z = (y[0] * 0.f + y[1] * 0.f) + (y[2] * 0.f + y[3] * 0.f);
    if (z != z) hi[g] = INFINITY;
  }
  KvqGroup gr[NG];
  if (values) {
#pragma unroll
    for (int g = 0; g < NG; ++g) gr[g] = kvq_group<BITS>(-row16_max(-lo[g]), row16_max(hi[g]));
  } else {
    float l = lo[0], m = hi[0];
#pragma unroll
    for (int g = 1; g < NG; ++g) {
      l = fminf(l, lo[g]);
      m = fmaxf(m, hi[g]);
    }
    l = fminf(l, dpp_f<Q35_DPP_QUAD_XOR1>(l)); m = fmaxf(m, dpp_f<Q35_DPP_QUAD_XOR1>(m));
    l = fminf(l, dpp_f<Q35_DPP_QUAD_XOR2>(l)); m = fmaxf(m, dpp_f<Q35_DPP_QUAD_XOR2>(m));
    if (E < 16) { l = fminf(l, dpp_f<Q35_DPP_ROW_HALF_MIRROR>(l)); m = fmaxf(m, dpp_f<Q35_DPP_ROW_HALF_MIRROR>(m)); }
    if (E < 8) { l = fminf(l, dpp_f<Q35_DPP_ROW_MIRROR>(l)); m = fmaxf(m, dpp_f<Q35_DPP_ROW_MIRROR>(m)); }
    gr[0] = kvq_group<BITS>(l, m);
#pragma unroll
    for (int g = 1; g < NG; ++g) gr[g] = gr[0];
  }
  if (pos < 0 || pos >= C) return;  // never write outside the cache (after the lane exchanges)
  uint32_t o[(E * BITS + 31) / 32];
#pragma unroll
  for (int j = 0; j < (E * BITS + 31) / 32; ++j) o[j] = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e * BITS / 32] |= kvq_encode<BITS>(x[e], gr[e / 4]) << (e * BITS % 32);
  uint8_t* dst = (values ? vq : kq) + ((size_t)bh * C + pos) * RB + c * (E * BITS / 8);
  if constexpr (E * BITS == 16) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)o[0];
  else if constexpr (E * BITS == 32) *reinterpret_cast<uint32_t*>(dst) = o[0];
  else if constexpr (E * BITS == 64) *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
  else *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
  uint32_t* pd = (values ? vp : kp) + (size_t)bh * NG * C + pos;
  if (values) {
    if (c < NG) {
      uint32_t word = gr[0].word;
#pragma unroll
      for (int g = 1; g < NG; ++g) word = c == g ? gr[g].word : word;
      pd[(size_t)c * C] = word;
    }
  } else if (c % (64 / E) == 0) {
    pd[(size_t)(c * E / 64) * C] = gr[0].word;
  }
}

// ---------------------------------------------------------------- read back
// The same 16 lanes a row: bf16(fma(code, step, low)), one rounding.
template <int E, int BITS>
__global__ __launch_bounds__(256) void kvq_read(const uint8_t* __restrict__ kq, const uint8_t* __restrict__ vq,
                                                const uint32_t* __restrict__ kp, const uint32_t* __restrict__ vp,
                                                uint16_t* __restrict__ k, uint16_t* __restrict__ v, int start,
                                                int L, int C, unsigned rows) {
  constexpr int NG = E / 4, RB = 2 * E * BITS;
  const unsigned row = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (row >= rows) return;
  const int c = threadIdx.x & 15;
  const unsigned bh = row / (unsigned)L, pos = start + row % (unsigned)L;
  const bool values = blockIdx.y != 0;
  const uint8_t* src = (values ? vq : kq) + ((size_t)bh * C + pos) * RB + c * (E * BITS / 8);
  const uint32_t* ps = (values ? vp : kp) + (size_t)bh * NG * C + pos;
  uint32_t w[(E * BITS + 31) / 32];
  if constexpr (E * BITS == 16) w[0] = *reinterpret_cast<const uint16_t*>(src);
  else if constexpr (E * BITS == 32) w[0] = *reinterpret_cast<const uint32_t*>(src);
  else if constexpr (E * BITS == 64) {
    const uint2 a = *reinterpret_cast<const uint2*>(src);
    w[0] = a.x; w[1] = a.y;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(src);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  }
  uint32_t p[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) p[g] = ps[(size_t)(values ? g : c * E / 64) * C];
  uint32_t o[E / 2];
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    const uint32_t pw = p[e / 4];
    const float st = bf_lo(pw), lw = bf_hi(pw);
    const float a = fmaf((float)kvq_code(w[e * BITS / 32], e % (32 / BITS), BITS), st, lw);
    const float d = fmaf((float)kvq_code(w[e * BITS / 32], e % (32 / BITS) + 1, BITS), st, lw);
    o[e / 2] = pack_bf2(a, d);
  }
  uint16_t* dst = (values ? v : k) + (size_t)row * (16 * E) + E * c;
  if constexpr (E == 4) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
  } else {
#pragma unroll
    for (int j = 0; j < E / 8; ++j)
      *reinterpret_cast<uint4*>(dst + 8 * j) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
  }
}

// ---------------------------------------------------------------- attention
// One wave a (batch, head, query row): lane l holds the V of its P = D / 64
// dims P l .., every key's score is reduced over the wave, online softmax in
// fp32. Row i of a sequence sees keys 0 .. start + i.
template <int P, int BITS>
__global__ __launch_bounds__(256) void kvq_attend_rows(
    const uint16_t* __restrict__ q, const uint8_t* __restrict__ kq, const uint8_t* __restrict__ vq,
    const uint32_t* __restrict__ kp, const uint32_t* __restrict__ vp, const long long* len_dev, int n_len,
    long long offset, const uint16_t* __restrict__ gate, long long gate_stride, float scale,
    uint16_t* __restrict__ out, int QH, int KVH, int L, int C, long long rows) {
  constexpr int D = 64 * P, NG = P, RB = D * BITS / 8;
  const int lane = threadIdx.x & 63;
  const long long wv = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (wv >= rows) return;
  const int i = L - 1 - (int)(wv % L);
  const int h = (int)(wv / L % QH);
  const int b = (int)(wv / L / QH);
  const size_t bh = (size_t)b * KVH + h / (QH / KVH);
  const long long at = (len_dev ? len_dev[n_len > 1 ? b : 0] : 0) + offset + i + 1;
  const int n = (int)(at < 0 ? 0 : at > C ? C : at);
  const uint16_t* qr = q + (((size_t)b * QH + h) * L + i) * D + P * lane;
  float qf[P], acc[P];
  int vg[P];
#pragma unroll
  for (int e = 0; e < P; ++e) {
    qf[e] = bf2f(qr[e]);
    acc[e] = 0.f;
    vg[e] = (P * lane + e) % (4 * P) / 4;
  }
  const int kg = P * lane / 64;
  const uint8_t* K = kq + bh * C * RB;
  const uint8_t* V = vq + bh * C * RB;
  const uint32_t* KP = kp + (bh * NG + kg) * C;
  const uint32_t* VP = vp + bh * NG * C;
  float m = -INFINITY, l = 0.f;
  auto code = [&](const uint8_t* base, int t, int d) {
    return BITS == 4 ? (float)((base[(size_t)t * RB + d / 2] >> (4 * (d & 1))) & 15) : (float)base[(size_t)t * RB + d];
  };
  for (int t = 0; t < n; ++t) {
    const uint32_t kw = KP[t];
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < P; ++e) s = fmaf(qf[e], fmaf(code(K, t, P * lane + e), bf_lo(kw), bf_hi(kw)), s);
    s = wave_sum(s) * scale;
    const float mn = fmaxf(m, s);
    const float corr = expf(m - mn), p = expf(s - mn);
    l = l * corr + p;
#pragma unroll
    for (int e = 0; e < P; ++e) {
      const uint32_t vw = VP[(size_t)vg[e] * C + t];
      acc[e] = fmaf(p, fmaf(code(V, t, P * lane + e), bf_lo(vw), bf_hi(vw)), acc[e] * corr);
    }
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < P; ++e) {
    const int d = P * lane + e;
    float o = n ? acc[e] / l : 0.f;  // a row without keys is zero
    if (gate) o *= sigmoid_f(bf2f(gate[b * gate_stride + (2 * h + 1) * D + d]));
    out[(((size_t)b * L + i) * QH + h) * D + d] = (uint16_t)f2bf(o);
  }
}

bool kvq_shape_ok(int B, int KVH, int L, int D, int bits, int C) {
  return B >= 0 && KVH > 0 && L >= 0 && (D == 64 || D == 128 || D == 256) && (bits == 4 || bits == 8) && C > 0 &&
         C % 32 == 0 && (long long)C * D * bits / 8 < (1ll << 31);
}

}  // namespace

extern "C" {

#define Q35_KVQ_BY_D(CALL)                                                          \
  do {                                                                              \
    if (bits == 4) {                                                                \
      if (D == 256) CALL(16, 4); else if (D == 128) CALL(8, 4); else CALL(4, 4);    \
    } else {                                                                        \
      if (D == 256) CALL(16, 8); else if (D == 128) CALL(8, 8); else CALL(4, 8);    \
    }                                                                               \
  } while (0)

int q35_kv_quantize(const void* k, long long k_sb, long long k_sh, long long k_sl, const void* v, long long v_sb,
                    long long v_sh, long long v_sl, void* kq, void* vq, void* kp, void* vp, const void* start_dev,
                    int n_start, long long start, int B, int KVH, int L, int D, int bits, int capacity,
                    hipStream_t stream) {
  Q35_CHECK_ARG(kvq_shape_ok(B, KVH, L, D, bits, capacity));
  if ((long long)B * L == 0) return 0;
  Q35_CHECK_ARG(!start_dev || n_start == 1 || n_start == B);
  Q35_CHECK_ARG(k && v && kq && vq && kp && vp && q35_aligned16(kq) && q35_aligned16(vq) && q35_aligned16(kp) &&
                q35_aligned16(vp));
  const bool wide = D > 64;
  Q35_CHECK_ARG(wide ? q35_aligned16(k) && q35_aligned16(v) : q35_aligned8(k) && q35_aligned8(v));
  Q35_CHECK_ARG((k_sb | k_sh | k_sl | v_sb | v_sh | v_sl) % (wide ? 8 : 4) == 0);
  const long long rows = (long long)B * KVH * L;
  Q35_CHECK_ARG(rows < (1ll << 31));
  const KvqSrc ks{(const uint16_t*)k, k_sb, k_sh, k_sl}, vs{(const uint16_t*)v, v_sb, v_sh, v_sl};
  const dim3 grid((unsigned)((rows + 15) / 16), 2);
#define Q35_CALL(E, BITS)                                                                                         \
  kvq_write<E, BITS><<<grid, 256, 0, stream>>>(ks, vs, (uint8_t*)kq, (uint8_t*)vq, (uint32_t*)kp, (uint32_t*)vp,   \
                                               (const long long*)start_dev, n_start, start, KVH, L, capacity,      \
                                               (unsigned)rows)
  Q35_KVQ_BY_D(Q35_CALL);
#undef Q35_CALL
  return q35_last_error();
}

int q35_kv_dequantize(const void* kq, const void* vq, const void* kp, const void* vp, void* k, void* v, int start,
                      int B, int KVH, int L, int D, int bits, int capacity, hipStream_t stream) {
  Q35_CHECK_ARG(kvq_shape_ok(B, KVH, L, D, bits, capacity));
  Q35_CHECK_ARG(start >= 0 && (long long)start + L <= capacity);
  if ((long long)B * L == 0) return 0;
  Q35_CHECK_ARG(kq && vq && kp && vp && k && v && q35_aligned16(kq) && q35_aligned16(vq) && q35_aligned16(kp) &&
                q35_aligned16(vp) && q35_aligned16(k) && q35_aligned16(v));
  const long long rows = (long long)B * KVH * L;
  Q35_CHECK_ARG(rows < (1ll << 31));
  const dim3 grid((unsigned)((rows + 15) / 16), 2);
#define Q35_CALL(E, BITS)                                                                                          \
  kvq_read<E, BITS><<<grid, 256, 0, stream>>>((const uint8_t*)kq, (const uint8_t*)vq, (const uint32_t*)kp,          \
                                              (const uint32_t*)vp, (uint16_t*)k, (uint16_t*)v, start, L, capacity,  \
                                              (unsigned)rows)
  Q35_KVQ_BY_D(Q35_CALL);
#undef Q35_CALL
  return q35_last_error();
}

long long q35_gqa_attention_kvq_workspace(int B, int QH, int KVH, int L, int D, int bits, int capacity) {
  if (!kvq_shape_ok(B, KVH, L, D, bits, capacity) || QH <= 0 || QH % KVH) return -1;
  return 0;
}

int q35_gqa_attention_kvq(const void* q, const void* kq, const void* vq, const void* kp, const void* vp,
                          const void* len_dev, int n_len, long long offset, const void* gate, long long gate_stride,
                          float scale, void* out, void* workspace, long long workspace_floats, int B, int QH, int KVH,
                          int L, int D, int bits, int capacity, hipStream_t stream) {
  Q35_CHECK_ARG(kvq_shape_ok(B, KVH, L, D, bits, capacity) && QH > 0 && QH % KVH == 0);
  if ((long long)B * L == 0) return 0;
  Q35_CHECK_ARG(!len_dev || n_len == 1 || n_len == B);
  Q35_CHECK_ARG(!gate || L == 1);
  Q35_CHECK_ARG(q && kq && vq && kp && vp && out && q35_aligned16(kq) && q35_aligned16(vq) && q35_aligned16(kp) &&
                q35_aligned16(vp) && q35_aligned16(q) && q35_aligned16(out) && q35_aligned8(gate));
  const long long rows = (long long)B * QH * L;
  Q35_CHECK_ARG(rows < (1ll << 31));
  const unsigned grid = (unsigned)((rows + 3) / 4);
#define Q35_CALL(E, BITS)                                                                                           \
  kvq_attend_rows<E / 4, BITS><<<grid, 256, 0, stream>>>(                                                           \
      (const uint16_t*)q, (const uint8_t*)kq, (const uint8_t*)vq, (const uint32_t*)kp, (const uint32_t*)vp,          \
      (const long long*)len_dev, n_len, offset, (const uint16_t*)gate, gate_stride, scale, (uint16_t*)out, QH, KVH,  \
      L, capacity, rows)
  Q35_KVQ_BY_D(Q35_CALL);
#undef Q35_CALL
  return q35_last_error();
}

}  // extern "C"
