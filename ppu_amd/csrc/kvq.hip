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
#include <cmath>
#include <type_traits>

#include "kvq.hpp"

namespace {

// Of two values, or a NaN if one is: the maxima that pass over a NaN would take an
// instruction more each.
Q35_DEV float kvq_most(float a, float b) { return __builtin_elementwise_maximum(a, b); }
Q35_DEV float kvq_least(float a, float b) { return __builtin_elementwise_minimum(a, b); }
template <int CTRL>
Q35_DEV float kvq_dpp(float v) {  // every lane has a source
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}

// The code of xh = x / 2 in a group with lh = low / 2 and sh = step / 2 from c, the
// code or one next to it: halves, as x - low may pass the fp32 range; halving and
// (code +- 1/2) * sh (at most 17 bits) are exact, and so is the error e of s = xh -
// lh, so the borders are compared in the real numbers.
Q35_DEV float kvq_exact_code(float xh, float lh, float sh, float c) {
  const float s = xh - lh;
  const float bb = s - xh;
  const float e = (xh - (s - bb)) + (-lh - bb);
  const bool odd = ((int)c & 1) != 0;
  const float hi = (c + 0.5f) * sh, lo = (c - 0.5f) * sh;
  if (s > hi || (s == hi && (e > 0.f || (e == 0.f && odd)))) c += 1.f;
  else if (s < lo || (s == lo && (e < 0.f || (e == 0.f && odd)))) c -= 1.f;
  return c;
}

// Greatest - low over T / 2, correctly rounded: a product with the constant's
// reciprocal and one correction by the remainder (checked for all 2^23 mantissas
// of both constants), above the range where the remainder would be inexact.
template <int BITS>
Q35_DEV float kvq_step(float r) {
  constexpr float H = BITS == 4 ? 7.5f : 127.5f, I = 1.0f / H;
  const float q = r * I;
  float v = fmaf(fmaf(-q, H, r), I, q);
  if (r < 1.0e-25f) v = r / H;
  return v;
}
// One group's step and low as the stored word, and its halves and reciprocal.
struct KvqGroup {
  uint32_t word;
  float lh, sh, inv;  // low / 2, step / 2 and 2 / step; inv NaN for a group that is
                      // not finite or whose step is too small for a reciprocal
};
template <int BITS>
Q35_DEV KvqGroup kvq_group(float lo, float hi) {
  KvqGroup g;
  const bool finite = lo > -INFINITY && hi < INFINITY;
  const uint32_t step = finite ? f2bf(kvq_step<BITS>(hi * 0.5f - lo * 0.5f)) : 0x7fc0u;
  g.word = step | (finite ? __float_as_uint(lo) & 0xffff0000u : 0x7fc00000u);
  g.lh = finite ? lo * 0.5f : 0.f;
  g.sh = finite ? bf2f(step) * 0.5f : 0.f;
  g.inv = g.sh >= 1.0e-30f ? __builtin_amdgcn_rcpf(g.sh) : finite && g.sh == 0.f ? 0.f : __builtin_nanf("");
  return g;
}
// The codes of E values, four of a group in turn. c, the whole number nearest to
// (x - low) / step as computed (off by less than 2^-21 of itself, 2^-13 at most), is
// the code or next to it, and the remainder is below half a step by more than its
// own error (2^-16 of a step) unless x lies on or next to the border of two codes:
// about one of 500 values does, on it, as bf16 values and steps have few bits. Those
// are looked at exactly, each in a branch of its own: with all of a lane's in one a
// write of 100003 tokens took 134 us.
template <int E, int BITS>
Q35_DEV void kvq_codes(const float (&x)[E], const KvqGroup (&g)[E / 4], uint32_t (&o)[(E * BITS + 31) / 32]) {
  constexpr float T = BITS == 4 ? 15.f : 255.f, NEAR = 0.5f - 0x1p-12f;
  float c[E], rest[E];
  bool far = true;
#pragma unroll
  for (int q = 0; q < E / 4; ++q) {
    const KvqGroup& y = g[q];
#pragma unroll
    for (int e = 4 * q; e < 4 * q + 4; ++e) {
      const float d = fmaf(x[e], 0.5f, -y.lh);
      c[e] = rintf(d * y.inv);
      rest[e] = fabsf(fmaf(-c[e], y.sh, d));
    }
    const float most = kvq_most(kvq_most(rest[4 * q], rest[4 * q + 1]), kvq_most(rest[4 * q + 2], rest[4 * q + 3]));
    far &= most <= y.sh * NEAR;  // not where it is NaN
  }
  if (!far) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const KvqGroup& y = g[e / 4];
      if (!(rest[e] <= y.sh * NEAR)) {
        if (!(y.inv > 0.f))  // a step below 2^-98, or none
          c[e] = y.sh > 0.f ? rintf((x[e] * 0.5f - y.lh) * 0x1p80f * __builtin_amdgcn_rcpf(y.sh * 0x1p80f)) : 0.f;
        if (y.sh > 0.f) c[e] = fmaxf(kvq_exact_code(x[e] * 0.5f, y.lh, y.sh, c[e]), 0.f);
      }
    }
  }
  // a step rounded down leaves up to 255.5 steps of 255, but 15.03 of 15
  if (BITS == 8) {
#pragma unroll
    for (int e = 0; e < E; ++e) c[e] = fminf(c[e], T);
  }
  // packed in fp32, where up to 24 bits are exact
  constexpr int N = 16 / BITS;  // codes of 16 bits
  constexpr float S = BITS == 4 ? 16.f : 256.f;
#pragma unroll
  for (int j = 0; j < (E * BITS + 31) / 32; ++j) {
    uint32_t half[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if ((2 * j + h) * N < E) {
        float v = c[(2 * j + h) * N + N - 1];
#pragma unroll
        for (int e = N - 2; e >= 0; --e) v = fmaf(v, S, c[(2 * j + h) * N + e]);
        half[h] = (uint32_t)v;
      }
    o[j] = half[0] | half[1] << 16;
  }
}

// ------------------------------------------------------------------- write
// 16 lanes a row: lane c holds run c, dims E c .. E c + E - 1 (E = D / 16). A
// key group is 64 / E lanes wide, a value group 4 dims of all 16 lanes. The heads'
// keys and values (blockIdx.y even and odd) read 2 D bytes and write D * bits / 8 +
// 4 D / 64 a row. 100003 tokens of 2 heads of 256 in 4 bits (262 MB) take 63 us, 4.1
// TB/s: bound by vector instructions, some 24 a value in all, so a lane of a quad
// works out the step of one group of values and the others take it from there
// (with each lane doing all, row and head from divisions and rounded divisions for
// the codes it was 83 us); one token takes a launch, 2.8 us.
struct KvqSrc {
  const uint16_t* p;
  long long sb, sh, sl;  // strides of batch, head, token in elements
};
template <int E, int BITS>
__global__ __launch_bounds__(256) void kvq_write(const KvqSrc ks, const KvqSrc vs, uint8_t* __restrict__ kq,
                                                 uint8_t* __restrict__ vq, uint32_t* __restrict__ kp,
                                                 uint32_t* __restrict__ vp, const long long* start_dev,
                                                 int n_start, long long start, int KVH, int L, int C) {
  constexpr int NG = E / 4, RB = 2 * E * BITS;  // groups, bytes of a packed row
  const unsigned t = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (t >= (unsigned)L) return;
  const int c = threadIdx.x & 15;
  const unsigned b = blockIdx.z, h = blockIdx.y >> 1, bh = b * KVH + h;
  const long long pos = (start_dev ? start_dev[n_start > 1 ? b : 0] : 0) + start + t;
  const bool values = blockIdx.y & 1;
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
  // Least and greatest value of 4 dims; a NaN stays one.
  float lo[NG], hi[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float* y = x + 4 * g;
    lo[g] = kvq_least(kvq_least(y[0], y[1]), kvq_least(y[2], y[3]));
    hi[g] = kvq_most(kvq_most(y[0], y[1]), kvq_most(y[2], y[3]));
  }
  KvqGroup own, gr[NG];  // the lane's own group of values is number c % NG: its share of the work
  if (values) {
    const auto exchange = [&](float (&v)[NG], auto pick) {  // of group c % NG
      float r[NG / 2 + 1] = {v[0]};
      if constexpr (NG == 1) {
        r[0] = pick(r[0], kvq_dpp<Q35_DPP_QUAD_XOR1>(r[0]));
      } else {
#pragma unroll
        for (int j = 0; j < NG / 2; ++j) {
          const float keep = c & 1 ? v[2 * j + 1] : v[2 * j], give = c & 1 ? v[2 * j] : v[2 * j + 1];
          r[j] = pick(keep, kvq_dpp<Q35_DPP_QUAD_XOR1>(give));
        }
      }
      if constexpr (NG == 4) {
        const float keep = c & 2 ? r[1] : r[0], give = c & 2 ? r[0] : r[1];
        r[0] = pick(keep, kvq_dpp<Q35_DPP_QUAD_XOR2>(give));
      } else {
        r[0] = pick(r[0], kvq_dpp<Q35_DPP_QUAD_XOR2>(r[0]));
      }
      r[0] = pick(r[0], kvq_dpp<0x124>(r[0]));  // row_ror:4
      return pick(r[0], kvq_dpp<0x128>(r[0]));  // row_ror:8
    };
    own = kvq_group<BITS>(exchange(lo, [](float p, float q) { return kvq_least(p, q); }),
                          exchange(hi, [](float p, float q) { return kvq_most(p, q); }));
    gr[0] = own;
    const auto from = [&](auto g) {  // lane g of the quad
      constexpr int CTRL = 0x55 * decltype(g)::value;
      gr[decltype(g)::value] = {0, kvq_dpp<CTRL>(own.lh), kvq_dpp<CTRL>(own.sh), kvq_dpp<CTRL>(own.inv)};
    };
    if constexpr (NG > 1) {
      from(std::integral_constant<int, 0>());
      from(std::integral_constant<int, 1>());
    }
    if constexpr (NG > 2) {
      from(std::integral_constant<int, 2>());
      from(std::integral_constant<int, 3>());
    }
  } else {
    float l = lo[0], m = hi[0];
#pragma unroll
    for (int g = 1; g < NG; ++g) {
      l = kvq_least(l, lo[g]);
      m = kvq_most(m, hi[g]);
    }
    l = kvq_least(l, kvq_dpp<Q35_DPP_QUAD_XOR1>(l)); m = kvq_most(m, kvq_dpp<Q35_DPP_QUAD_XOR1>(m));
    l = kvq_least(l, kvq_dpp<Q35_DPP_QUAD_XOR2>(l)); m = kvq_most(m, kvq_dpp<Q35_DPP_QUAD_XOR2>(m));
    if (E < 16) { l = kvq_least(l, kvq_dpp<Q35_DPP_ROW_HALF_MIRROR>(l)); m = kvq_most(m, kvq_dpp<Q35_DPP_ROW_HALF_MIRROR>(m)); }
    if (E < 8) { l = kvq_least(l, kvq_dpp<Q35_DPP_ROW_MIRROR>(l)); m = kvq_most(m, kvq_dpp<Q35_DPP_ROW_MIRROR>(m)); }
    own = kvq_group<BITS>(l, m);
#pragma unroll
    for (int g = 0; g < NG; ++g) gr[g] = own;
  }
  if (pos < 0 || pos >= C) return;  // never write outside the cache (after the lane exchanges)
  uint32_t o[(E * BITS + 31) / 32];
  kvq_codes<E, BITS>(x, gr, o);
  uint8_t* dst = (values ? vq : kq) + ((size_t)bh * C + pos) * RB + c * (E * BITS / 8);
  if constexpr (E * BITS == 16) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)o[0];
  else if constexpr (E * BITS == 32) *reinterpret_cast<uint32_t*>(dst) = o[0];
  else if constexpr (E * BITS == 64) *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
  else *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
  uint32_t* pd = (values ? vp : kp) + (size_t)bh * NG * C + pos;
  if (values) {
    if (c < NG) pd[(size_t)c * C] = own.word;
  } else if (c % (64 / E) == 0) {
    pd[(size_t)(c * E / 64) * C] = own.word;
  }
}

// ------------------------------------------------- attention of a few rows
// The query rows of one KV head, G = QH / KVH heads x L tokens, in blocks of HP
// rows; a workgroup takes one block and every S-th piece of NW x 32 keys, a
// wave one tile of 32 keys of each piece. Products are transposed, keys or dims
// as the rows of v_mfma_f32_16x16x32_bf16 and query rows as its columns, and a
// column is a pair (query row, group): the 16 columns are HP rows x GT of the
// NG groups, CT = NG / GT column tiles in all. A lane then needs one step and
// one low per key, its own group's:
//   S^T[key, (row, group)] = step (K' Q^T) + low sum(q), K' = the codes and Q
//     zero outside the column's group; the groups' parts are added over GT
//     neighbouring lanes. The codes are taken as fp8 as they stand: the byte 0000
//     cccc is c 2^-9 in e4m3, so two ands and a shift make 8 operands of a word
//     (of 8-bit codes the two halves, 16 apart). Q times a power of two of its
//     row (its greatest in [2^7, 2^8)) is the sum of two fp8 values, exact but
//     for values below 2^-9 of the greatest, which are off by 2^-17 of it at
//     most; for the low halves of 8-bit codes it is 2^-4 of that, so 2^-5 and
//     2^-13, of at most 15 steps where the group has 255.
//   O^T[dim, (row, group)] += V' A^T, A = p step of the column's group as bf16
//     hi + lo (error below 2^-16: one bf16 would be off by 2^-8 of the group's
//     range, whatever the value), and p low in fp32 beside it; V' = 16 + code in
//     bf16 by one shift and one and-or for two 4-bit codes, 8-bit codes are
//     converted; row c of V' product i is dim (D / 16) c + i of every run, all
//     in group i / 4. The offset's sum over A is one more product with constant
//     rows.
// P never leaves its lane: the C layout of S^T (lane: 4 keys of a column) is the
// B operand of O^T when the 32 keys of a step are taken in the order {4 kg .. 4
// kg + 3, 16 + 4 kg ..}. Codes are exact.
//
// Bound by memory in a long cache, by latency in a short one (8/2 heads of 256, 4
// bits: 131071 tokens 22 us with the merge, of which a plain read of the 75 MB in a
// launch is 13.6 and the merge 4.5; without any arithmetic the same copies take 20;
// 1088 tokens 7.9, two launches with one round trip for the length and one for the
// tile). fp8 products run at the rate of bf16 ones here, what they save is the
// conversion. Copies straight into LDS need no registers, so two tiles a wave are
// in flight beside the sums; loads into registers waited for each other.
//
// The running maximum m (log2 units) moves only when a tile passes it by 8, so O
// is rescaled a few times a row. Tiles are dealt in turn, so any valid length
// spreads over all splits. Keys past a row's end are masked in S and their step
// and low set to zero, whatever their params hold.
template <int D, int BITS, int HP>
struct KvqFew {
  static constexpr int NG = D / 64, GT = NG < 16 / HP ? NG : 16 / HP, CT = NG / GT, NW = 4;
  static constexpr int KW = BITS / 2;                   // words of a lane's 16 dims of a key group
  static constexpr int RB = D * BITS / 8;               // bytes of a packed row
  static constexpr int RUN = RB / 16;                   // bytes of a run
  static constexpr int VR = RUN < 4 ? 1 : RUN / 4;      // words that hold it
  static constexpr int NK = RB / 32;                    // 1 KiB copies of a tile's keys (and of its values)
  static constexpr int NI = 2 * NK + 1;                 // copies of a tile
  static constexpr int STAGE = 1024 * NI;               // keys, values, params (2 NG lines of 128 bytes)
  static constexpr int RING = 2 * STAGE;                // a wave's two tiles
  static constexpr int QB = HP * D * 2;                 // bytes of a block's queries
  static constexpr int REC = HP * (D + 2);              // floats of a split's record
  static constexpr int WAVES = BITS == 4 && !(D == 256 && HP > 8) ? 2 : 1;  // waves a SIMD, by registers
  struct Tile {
    uint32_t k[2][NG][KW], v[8][VR], kp[2][CT][4], vp[2][CT][4];
  };
};

// One wave instruction of a copy: lane i's 16 bytes at p to LDS bytes [lds + 16
// i, +16).
Q35_DEV void kvq_copy(uint32_t lds, const uint8_t* p) {
  asm volatile("global_load_lds_dwordx4 %0, off" : : "v"(p), "{m0}"(lds) : "memory");
}
// The slot of chunk 0 of a key row of RB bytes in LDS; the place of value row r.
template <int RB>
Q35_DEV uint32_t kvq_swz(uint32_t row) { return row / (256 / RB) % (RB / 16); }
template <int RB>
Q35_DEV uint32_t kvq_turn(uint32_t r) {
  if (RB == 32) return r;
  if (RB == 64) return (r & 17) | ((r & 6) << 1) | ((r >> 2) & 2);
  return (r & 16) | ((r & 3) << 2) | ((r >> 2) & 3);
}

// Two 4-bit codes (nibble i of each half of w) as 16 + code in bf16.
// One v_and_or_b32 takes its constants from registers, one of them a vector's.
struct KvqMask {
  uint32_t mask, off;
};
Q35_DEV KvqMask kvq_mask() {
  KvqMask c{0x00780078u, 0x41804180u};
  asm("" : "+s"(c.mask), "+v"(c.off));
  return c;
}
template <int I>
Q35_DEV uint32_t kvq_pair4(uint32_t w, const KvqMask& c) {
  const uint32_t t = I == 0 ? w << 3 : w >> (4 * I - 3);
  return (t & c.mask) | c.off;
}
// Byte i of two words as bf16.
template <int I>
Q35_DEV uint32_t kvq_pair8(uint32_t w0, uint32_t w1) {
  const float a = (float)((w0 >> (8 * I)) & 255u), b = (float)((w1 >> (8 * I)) & 255u);
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

Q35_DEV float kvq_xor16_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
Q35_DEV float kvq_xor16_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Over the 4 lanes of a column.
Q35_DEV float kvq_col_max(float v) { return half_max(kvq_xor16_max(v)); }
Q35_DEV float kvq_col_sum(float v) { return half_sum(kvq_xor16_sum(v)); }

// Four values as fp8 (e4m3) bytes; byte i back.
Q35_DEV uint32_t kvq_fp8(const float (&y)[4]) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
}
Q35_DEV float kvq_from_fp8(uint32_t w, int i) {
  return i == 0   ? __builtin_amdgcn_cvt_f32_fp8((int)w, 0)
         : i == 1 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 1)
         : i == 2 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 2)
                  : __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
}
Q35_DEV q35_f32x4 mfma8(const q35_u32x2 a, const q35_u32x2 b, q35_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(__builtin_bit_cast(long, a), __builtin_bit_cast(long, b), c, 0, 0, 0);
}
Q35_DEV q35_f32x4 mfma16(const q35_u32x4 a, const q35_u32x4 b, q35_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(q35_bf16x8, a), __builtin_bit_cast(q35_bf16x8, b),
                                                 c, 0, 0, 0);
}

// Sequences of unequal lengths share the workgroups of a KV head (at most 64
// sequences, lane i holds sequence i): sequence i takes s_i = max(1, floor(share
// p_i / sum p)) of them, p_i its pieces of 128 keys, at numbers first_i .. first_i
// + s_i - 1, so that every workgroup has about as many pieces: at most share + B
// in all, those that are left over last in the launch, as a launch's workgroups
// are dealt to the CUs in order. With splits fixed a sequence, 60000 and 15 x 1000
// tokens (8 KV heads of 128) took 99 us.
constexpr int kKvqShared = 64;
struct KvqShares {
  long long start;
  int s, first;
};
Q35_DEV KvqShares kvq_shares(const KvqShape& a, int lane) {
  KvqShares v;
  v.start = (lane < a.B ? a.len[lane] : 0) + a.offset;
  const int p = lane < a.B ? (kvq_limit(a, v.start, a.L - 1) + 127) / 128 : 0;
  const int total = wave_sum_i32(p);
  v.s = p ? max(min(min(p, a.share), (int)((float)p * (float)a.share / (float)total)), 1) : 0;
  int incl = v.s;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
  v.first = incl - v.s;
  return v;
}
Q35_DEV long long kvq_lane64(long long v, int lane) {
  return (long long)(((unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
                     (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
}

template <int D, int BITS, int HP>
__global__ __launch_bounds__(256, (KvqFew<D, BITS, HP>::WAVES)) void kvq_few(const KvqArgs a) {
  using F = KvqFew<D, BITS, HP>;
  using Tile = typename F::Tile;
  constexpr int NG = F::NG, GT = F::GT, CT = F::CT, NW = F::NW, KW = F::KW, VR = F::VR, NT = D / 16;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int c16 = lane & 15, kg = lane >> 4, hr = c16 / GT, gl = c16 % GT;
  // Blocks of the same keys (a unit: split of a KV head) are 8 workgroups apart,
  // on one XCD and its L2, and next in turn; units go round the XCDs. Fewer than 8
  // units go round themselves, each on its share of the XCDs (800 rows of 512 keys on
  // one KV head of 256, 4 units: 15.8 us, on 4 XCDs alone 23.2).
  int split = blockIdx.x, blk = 0, kvh = blockIdx.y, b = blockIdx.z;
  if (a.blocks > 1) {
    const int round = min(a.B * a.KVH * a.splits, 8);
    const int x = (int)blockIdx.x / round, unit = x / a.blocks * round + (int)blockIdx.x % round;
    blk = x % a.blocks;
    const int h = unit / a.splits;
    split = unit - h * a.splits;
    b = h / a.KVH;
    kvh = h - b * a.KVH;
    if (b >= a.B) return;
  }
  int splits = a.splits, rec_at;
  long long start;
  if (a.share) {
    split = (int)blockIdx.x / a.KVH;
    kvh = (int)blockIdx.x - split * a.KVH;
    const KvqShares v = kvq_shares(a, lane);
    const uint64_t mine = __ballot(split >= v.first && split < v.first + v.s);
    if (!mine) return;
    b = __ffsll((long long)mine) - 1;
    rec_at = (a.share + a.B) * kvh + split;
    split -= __builtin_amdgcn_readlane(v.first, b);
    splits = __builtin_amdgcn_readlane(v.s, b);
    start = kvq_lane64(v.start, b);
  } else {
    rec_at = ((b * a.KVH + kvh) * a.blocks + blk) * splits + split;
    start = kvq_start(a, b);
  }
  const int bh = b * a.KVH + kvh;
  const int G = a.G, R = G * a.L;

  __shared__ alignas(1024) uint8_t lds[NW * F::RING + F::QB];
  __shared__ float ml_s[NW][HP][2];
  uint8_t* ring = lds + w * F::RING;
  uint8_t* q_raw = lds + NW * F::RING;
  const uint32_t ring0 = __builtin_amdgcn_readfirstlane(lds_offset(ring));

  // ---- queries of the block into LDS, wave w's share 1 KiB at a time
  const int row0 = blk * HP;
#pragma unroll
  for (int z = 0; z < (F::QB + 1024 * NW - 1) / (1024 * NW); ++z) {
    const int at = 1024 * (w + NW * z);
    if (at < F::QB) {
      const int r = min(row0 + (at + 16 * lane) / (2 * D), R - 1), i = kvq_token(a, r);
      kvq_copy(__builtin_amdgcn_readfirstlane(lds_offset(q_raw + at)),
               (const uint8_t*)(a.q + (((size_t)bh * G + (r - i * G)) * a.L + i) * D) +
                   (at + 16 * lane) % (2 * D));
    }
  }

  // ---- a tile: every copy takes 1 KiB in whole rows. Key rows keep their
  // order, chunk c of 16 bytes at slot c ^ swz(row), so the 16 rows of a
  // fragment read fall on distinct bank groups. The value rows that a read
  // takes, 4 apart, are put next to each other, 4 x 4 transposed within 16 (row
  // r holds token turn(r)), as far as whole 128-byte lines stay together.
  constexpr int RB = F::RB, CPR = RB / 16;
  const uint8_t* K = a.kq + (size_t)bh * a.C * RB;
  const uint8_t* V = a.vq + (size_t)bh * a.C * RB;
  uint32_t k_at[F::NK], v_at[F::NK];
#pragma unroll
  for (int z = 0; z < F::NK; ++z) {
    const uint32_t row = (64 * z + lane) / CPR, slot = lane % CPR;
    k_at[z] = row * RB + 16 * (slot ^ kvq_swz<RB>(row));
    v_at[z] = kvq_turn<RB>(row) * RB + 16 * slot;
  }
  const uint8_t* p_at;
  {
    const int i = lane % (16 * NG), g = i / 8 % NG;
    p_at = (const uint8_t*)((i < 8 * NG ? a.kp : a.vp) + ((size_t)bh * NG + g) * a.C) + 16 * (i % 8);
  }
  auto issue = [&](int tile, int stage) {
    const uint32_t to = ring0 + F::STAGE * stage;
    const uint8_t *kb = K + (size_t)tile * (32 * RB), *vb = V + (size_t)tile * (32 * RB);
#pragma unroll
    for (int z = 0; z < F::NK; ++z) dma16(to + 1024 * z, kb, k_at[z]);
    kvq_copy(to + 2048 * F::NK, p_at + (size_t)tile * 128);
#pragma unroll
    for (int z = 0; z < F::NK; ++z) dma16(to + 1024 * (F::NK + z), vb, v_at[z]);
  };
  const int limit = kvq_limit(a, start, kvq_token(a, min(row0 + hr, R - 1)));
  const int least = kvq_limit(a, start, kvq_token(a, row0));
  const int n_max = kvq_limit(a, start, kvq_token(a, min(row0 + HP, R) - 1));
  const int n_tiles = (n_max + 31) / 32;
  const int stride = splits * NW;
  int tile = split * NW + w;
  if (tile < n_tiles) issue(tile, 0);
  if (tile + stride < n_tiles) issue(tile + stride, 1);

  // ---- fragment addresses in a stage
  uint32_t k_rd[2], v_rd, p_rd;
#pragma unroll
  for (int tt = 0; tt < 2; ++tt) k_rd[tt] = (16 * tt + c16) * RB;
  v_rd = 1024 * F::NK + kg * (RB == 32 ? 4 : RB == 64 ? 2 : 1) * RB + F::RUN * c16;
  p_rd = 2048 * F::NK + 128 * gl + 16 * kg;
  auto fetch_k = [&](Tile& t, int stage) {
    const uint8_t* s = ring + F::STAGE * stage;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        // the lane's 16 dims: bytes 4 KW (4 g + kg)
        const uint32_t c = KW == 4 ? 4 * g + kg : 2 * g + (kg >> 1);
        const uint8_t* p = s + k_rd[tt] + 16 * (c ^ kvq_swz<RB>(16 * tt + c16)) + (KW == 4 ? 0 : 8 * (kg & 1));
        if constexpr (KW == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(p);
          t.k[tt][g][0] = x.x; t.k[tt][g][1] = x.y;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(p);
          t.k[tt][g][0] = x.x; t.k[tt][g][1] = x.y; t.k[tt][g][2] = x.z; t.k[tt][g][3] = x.w;
        }
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const uint4 x = *reinterpret_cast<const uint4*>(s + p_rd + 128 * GT * ct + 64 * tt);
        t.kp[tt][ct][0] = x.x; t.kp[tt][ct][1] = x.y; t.kp[tt][ct][2] = x.z; t.kp[tt][ct][3] = x.w;
      }
    }
  };
  auto fetch_v = [&](Tile& t, int stage) {
    const uint8_t* s = ring + F::STAGE * stage;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const uint4 y = *reinterpret_cast<const uint4*>(s + p_rd + 128 * (NG + GT * ct) + 64 * tt);
        t.vp[tt][ct][0] = y.x; t.vp[tt][ct][1] = y.y; t.vp[tt][ct][2] = y.z; t.vp[tt][ct][3] = y.w;
      }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // token 16 tt + 4 kg + i
      const int i = j & 3, at = RB == 32 ? i : RB == 64 ? 8 * (i >> 1) + (i & 1) : 4 * i;
      const uint8_t* p = s + v_rd + (16 * (j >> 2) + at) * RB;
      if constexpr (F::RUN == 2) t.v[j][0] = *reinterpret_cast<const uint16_t*>(p);
      else if constexpr (F::RUN == 4) t.v[j][0] = *reinterpret_cast<const uint32_t*>(p);
      else if constexpr (F::RUN == 8) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        t.v[j][0] = x.x; t.v[j][1] = x.y;
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        t.v[j][0] = x.x; t.v[j][1] = x.y; t.v[j][2] = x.z; t.v[j][3] = x.w;
      }
    }
  };

  // ---- Q of the lane's row: dims 64 g + 16 kg + 8 h .. + 7 in step (g, h), zero
  // outside the column's group, in the order of the codes' bytes. The queries
  // were copied first: they are there when at most the tiles are not.
  if (tile + stride < n_tiles) wait_vm<2 * F::NI>();
  else if (tile < n_tiles) wait_vm<F::NI>();
  else wait_vm<0>();
  __syncthreads();
  constexpr int P = BITS == 4 ? 2 : 4;
  q35_u32x2 qf[NG][2][P];
  float qs[CT], back;  // sums over whole groups; what brings S back
  {
    const uint8_t* qp = q_raw + hr * (2 * D) + 32 * kg;
    const uint32_t neg = a.scale < 0.f ? 0x80008000u : 0u;
    float x[CT][2][8], top = 0.f;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 y = *reinterpret_cast<const uint4*>(qp + 128 * (ct * GT + gl) + 16 * h);
        y.x ^= neg; y.y ^= neg; y.z ^= neg; y.w ^= neg;
        unpack8(y, x[ct][h]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum += x[ct][h][e];
          top = fmaxf(top, fabsf(x[ct][h][e]));
        }
      }
      qs[ct] = kvq_col_sum(sum);
    }
    top = kvq_col_max(top);
    if constexpr (GT > 1) top = fmaxf(top, dpp_f<Q35_DPP_QUAD_XOR1>(top));
    if constexpr (GT > 2) top = fmaxf(top, dpp_f<Q35_DPP_QUAD_XOR2>(top));
    const int shift = kvq_shift(top, BITS == 4 ? 7 : 3);
    const float up = exp2_int(shift);
    back = exp2_int(-shift);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      qs[ct] *= up * (1.0f / 512.0f);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < P / 2; ++n) {
          const float f = n ? 16.f * up : up;
          q35_u32x2 own[2];
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = x[ct][h][BITS == 4 ? 2 * e + v : 4 * v + e] * f;
            own[0][v] = kvq_fp8(y);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] -= kvq_from_fp8(own[0][v], e);
            own[1][v] = kvq_fp8(y);
          }
#pragma unroll
          for (int g = 0; g < GT; ++g)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              qf[ct * GT + g][h][2 * n][v] = gl == g ? own[0][v] : 0u;
              qf[ct * GT + g][h][2 * n + 1][v] = gl == g ? own[1][v] : 0u;
            }
        }
    }
  }
  // log2 e |scale|, the sign in Q; never 0, which would make NaN of a masked -inf
  const float c2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f * 512.f * back, 1.0e-37f);
  const KvqMask cm = kvq_mask();
  q35_f32x4 o[NT], cnt[CT];
  float cs[CT];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    cnt[ct] = {0.f, 0.f, 0.f, 0.f};
    cs[ct] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const uint32_t offs = 0xc180c180u;  // bf16 -16
  const q35_u32x4 ones = {offs, offs, offs, offs};

  auto step = [&](int tile, int stage) {
    const int key0 = 32 * tile;
    Tile t;
    fetch_k(t, stage);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      q35_f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int x = 0; x < GT; ++x) {
        const int g = ct * GT + x;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) {
            if constexpr (BITS == 4) {
              const uint32_t kw = t.k[tt][g][h];
              const q35_u32x2 kf = {kw & 0x0f0f0f0fu, (kw >> 4) & 0x0f0f0f0fu};
              acc[tt] = mfma8(kf, qf[g][h][0], acc[tt]);
              acc[tt] = mfma8(kf, qf[g][h][1], acc[tt]);
            } else {
              const uint32_t k0 = t.k[tt][g][2 * h], k1 = t.k[tt][g][2 * h + 1];
              const q35_u32x2 lo = {k0 & 0x0f0f0f0fu, k1 & 0x0f0f0f0fu};
              const q35_u32x2 hi = {(k0 >> 4) & 0x0f0f0f0fu, (k1 >> 4) & 0x0f0f0f0fu};
              acc[tt] = mfma8(lo, qf[g][h][0], acc[tt]);
              acc[tt] = mfma8(lo, qf[g][h][1], acc[tt]);
              acc[tt] = mfma8(hi, qf[g][h][2], acc[tt]);
              acc[tt] = mfma8(hi, qf[g][h][3], acc[tt]);
            }
          }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t pw = t.kp[j >> 2][ct][j & 3];
        const float st = bf_lo(pw);
        s[j] = fmaf(st, acc[j >> 2][j & 3], fmaf(bf_hi(pw), qs[ct], s[j]));
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (GT > 1) s[j] += dpp_f<Q35_DPP_QUAD_XOR1>(s[j]);
      if constexpr (GT > 2) s[j] += dpp_f<Q35_DPP_QUAD_XOR2>(s[j]);
    }
    // the tile's last reads, and its place takes the copies of the tile after next
    Q35_PIN();
    fetch_v(t, stage);
    wait_lds();
    Q35_PIN();
    if (tile + 2 * stride < n_tiles) issue(tile + 2 * stride, stage);
    Q35_PIN();
    float vs[CT][8], vm[CT][8];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const uint32_t(&pw)[4] = t.vp[tt][ct];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          vs[ct][4 * tt + i] = bf_lo(pw[i]);
          vm[ct][4 * tt + i] = bf_hi(pw[i]);
        }
      }
    if (key0 + 32 > least) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = key0 + 16 * (j >> 2) + 4 * kg + (j & 3) < limit;
        s[j] = in ? s[j] : -INFINITY;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          vs[ct][j] = in ? vs[ct][j] : 0.f;
          vm[ct][j] = in ? vm[ct][j] : 0.f;
        }
      }
    }
    float mx = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mx = fmaxf(mx, s[j]);
    mx = kvq_col_max(mx) * c2;
    if (__ballot(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx);
      const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= corr;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= corr;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        cs[ct] *= corr;
        cnt[ct][0] *= corr;  // the other rows of cnt are copies, unused
      }
      m = mn;
    }
    const float ms = m == -INFINITY ? 0.f : m;  // a row without any key so far
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f(fmaf(s[j], c2, -ms));
      l += p[j];
    }
    q35_u32x4 af[CT], al[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = p[2 * e] * vs[ct][2 * e], y = p[2 * e + 1] * vs[ct][2 * e + 1];
        af[ct][e] = pack_bf2(x, y);
        al[ct][e] = pack_bf2(x - bf_lo(af[ct][e]), y - bf_hi(af[ct][e]));
        cs[ct] = fmaf(p[2 * e], vm[ct][2 * e], cs[ct]);
        cs[ct] = fmaf(p[2 * e + 1], vm[ct][2 * e + 1], cs[ct]);
      }
      if constexpr (BITS == 4) {
        cnt[ct] = mfma16(ones, af[ct], cnt[ct]);
        cnt[ct] = mfma16(ones, al[ct], cnt[ct]);
      }
    }
    // Four dims a turn (one group): the hi parts' products, then the lo parts'.
#pragma unroll
    for (int g = 0; g < NT / 4; ++g) {
      q35_u32x4 vf[4];
      if constexpr (BITS == 4) {
        const int x = g / 2;
        const uint32_t sel = g & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t h = __builtin_amdgcn_perm(t.v[2 * e + 1][x], t.v[2 * e][x], sel);
          vf[0][e] = kvq_pair4<0>(h, cm); vf[1][e] = kvq_pair4<1>(h, cm);
          vf[2][e] = kvq_pair4<2>(h, cm); vf[3][e] = kvq_pair4<3>(h, cm);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t v0 = t.v[2 * e][g], v1 = t.v[2 * e + 1][g];
          vf[0][e] = kvq_pair8<0>(v0, v1); vf[1][e] = kvq_pair8<1>(v0, v1);
          vf[2][e] = kvq_pair8<2>(v0, v1); vf[3][e] = kvq_pair8<3>(v0, v1);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) o[4 * g + i] = mfma16(vf[i], af[g / GT], o[4 * g + i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[4 * g + i] = mfma16(vf[i], al[g / GT], o[4 * g + i]);
    }
  };
  // Two tiles in flight.
  for (int stage = 0; tile < n_tiles; stage ^= 1) {
    if (tile + stride < n_tiles) wait_vm<F::NI>();
    else wait_vm<0>();
    asm volatile("" : : : "memory");
    Q35_PIN();
    step(tile, stage);
    Q35_PIN();
    tile += stride;
  }

  // The waves' sums meet in LDS, each in its own ring: row hr, dims (D / 16) (4
  // kg + e) + 4 g .. + 3 of the lane's groups g.
  static_assert(HP * D * 4 <= F::RING, "a wave's sums fit its ring");
  l = kvq_col_sum(l);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const float add = kvq_col_sum(cs[ct]) + cnt[ct][0];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        v[x] = o[4 * ct * GT + x][e];
#pragma unroll
        for (int g = 1; g < GT; ++g) v[x] = gl == g ? o[4 * (ct * GT + g) + x][e] : v[x];
        v[x] += add;
      }
      *reinterpret_cast<float4*>(ring + 4 * (hr * D + NT * (4 * kg + e) + 4 * (ct * GT + gl))) =
          make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  if (kg == 0 && gl == 0) {
    ml_s[w][hr][0] = m;
    ml_s[w][hr][1] = l;
  }
  __syncthreads();
  float* rec = a.part + (size_t)rec_at * F::REC;
  for (int x = threadIdx.x; x < HP * D / 4; x += 256) {
    const int h = x / (D / 4), d = 4 * (x % (D / 4));
    float mm = -INFINITY;
#pragma unroll
    for (int v = 0; v < NW; ++v) mm = fmaxf(mm, ml_s[v][h][0]);
    const float ms = mm == -INFINITY ? 0.f : mm;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float ll = 0.f;
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float f = __builtin_amdgcn_exp2f(ml_s[v][h][0] - ms);  // 0 for a wave without keys
      const float4 t = *reinterpret_cast<const float4*>(lds + v * F::RING + 4 * (h * D + d));
      sum.x = fmaf(t.x, f, sum.x); sum.y = fmaf(t.y, f, sum.y);
      sum.z = fmaf(t.z, f, sum.z); sum.w = fmaf(t.w, f, sum.w);
      ll = fmaf(ml_s[v][h][1], f, ll);
    }
    *reinterpret_cast<float4*>(rec + h * D + d) = sum;
    if (d == 0) *reinterpret_cast<float2*>(rec + HP * D + 2 * h) = make_float2(mm, ll);
  }
}

// Merge of the splits that had keys: o = sum_s o_s 2^(m_s - M) / sum_s l_s
// 2^(m_s - M), M = max m_s. One workgroup a query row and 64 dims, 16 threads of
// 4 dims by 16 parts of the splits, so a thread reads PER = splits / 16 records
// of at most 256. Bound by latency: all of a thread's reads are requested at once.
// PER by the number of splits, after 512 tokens 7.6 us in all, with 16 always 8.0.
constexpr int kKvqSplits = 256;
template <int D, int HP, int PER>
__global__ __launch_bounds__(256) void kvq_few_merge(const KvqMergeArgs a) {
  constexpr int NW = 4, REC = HP * (D + 2);
  const int t = threadIdx.x, part = t >> 4;
  const int r = blockIdx.x / (D / 64), d = 64 * (int)(blockIdx.x % (D / 64)) + 4 * (t & 15);
  const int kvh = blockIdx.y, b = blockIdx.z, bh = b * a.KVH + kvh, blk = r / HP, h = r % HP;
  // Requested together: a part's records, the thread's split's (m, l) and the
  // length that says which of them were written.
  const float* rec = a.part + (size_t)(bh * a.blocks + blk) * a.splits * REC;
  long long start;
  int splits = a.splits;
  if (a.share) {
    const KvqShares v = kvq_shares(a, t & 63);
    rec = a.part + (size_t)((a.share + a.B) * kvh + __builtin_amdgcn_readlane(v.first, b)) * REC;
    splits = max(__builtin_amdgcn_readlane(v.s, b), 1);
    start = kvq_lane64(v.start, b);
  } else {
    start = kvq_start(a, b);
  }
  const float2 raw = *reinterpret_cast<const float2*>(rec + (size_t)min(t, splits - 1) * REC + HP * D + 2 * h);
  float4 x[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j)
    x[j] = *reinterpret_cast<const float4*>(rec + (size_t)min(part + 16 * j, splits - 1) * REC + h * D + d);
  const int i = kvq_token(a, r), head = kvh * a.G + (r - i * a.G);
  const uint2 gate = a.gate ? *reinterpret_cast<const uint2*>(a.gate + (size_t)b * a.gate_stride + (2 * head + 1) * D + d)
                            : make_uint2(0, 0);
  const int n_max = kvq_limit(a, start, kvq_token(a, min(blk * HP + HP, a.G * a.L) - 1));
  const int n = min(splits, ((n_max + 31) / 32 + NW - 1) / NW);
  __shared__ float f_s[kKvqSplits], red_s[2][4];
  __shared__ float4 sum_s[16][16];
  const float m = t < n ? raw.x : -INFINITY, l = t < n ? raw.y : 0.f;
  const float mw = wave_max(m);
  if ((t & 63) == 0) red_s[0][t >> 6] = mw;
  __syncthreads();
  const float mm = fmaxf(fmaxf(red_s[0][0], red_s[0][1]), fmaxf(red_s[0][2], red_s[0][3]));
  const float f = __builtin_amdgcn_exp2f(m - (mm == -INFINITY ? 0.f : mm));
  f_s[t] = f;
  const float lw = wave_sum(l * f);
  if ((t & 63) == 0) red_s[1][t >> 6] = lw;
  __syncthreads();
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (part + 16 * j < n) {  // not a weight of 0: what was not written may be anything
      const float fs = f_s[part + 16 * j];
      sum.x = fmaf(x[j].x, fs, sum.x); sum.y = fmaf(x[j].y, fs, sum.y);
      sum.z = fmaf(x[j].z, fs, sum.z); sum.w = fmaf(x[j].w, fs, sum.w);
    }
  }
  sum_s[part][t & 15] = sum;
  __syncthreads();
  if (part) return;
#pragma unroll
  for (int v = 1; v < 16; ++v) {
    const float4 y = sum_s[v][t];
    sum.x += y.x; sum.y += y.y; sum.z += y.z; sum.w += y.w;
  }
  // a row without keys is zero
  const float inv = kvq_limit(a, start, i) ? 1.0f / ((red_s[1][0] + red_s[1][1]) + (red_s[1][2] + red_s[1][3])) : 0.f;
  float v[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
  if (a.gate) {
    v[0] *= sigmoid_f(bf_lo(gate.x)); v[1] *= sigmoid_f(bf_hi(gate.x));
    v[2] *= sigmoid_f(bf_lo(gate.y)); v[3] *= sigmoid_f(bf_hi(gate.y));
  }
  *reinterpret_cast<uint2*>(a.out + (((size_t)b * a.L + i) * (a.G * a.KVH) + head) * D + d) =
      make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
}

// Whether the rows of a KV head go to kvq_few, which reads and unpacks the keys
// once per block of rows, or to kvq_prompt, which unpacks them once into memory and
// has several launches: up to the rows at which unpacking a large cache pays, or
// little work in all, where a longer cache takes kvq_prompt longer to start (both
// borders fitted). Both ways, us (GPU time, 4 bits): 8/2 heads of 256, 512 keys: 512
// rows 18 / 23, 1024 31 / 24; 2048 keys: 512 32 / 36, 1024 44 / 38; 8192 keys: 256 39 /
// 55, 512 57 / 53; 32768 keys: 128 54 / 79, 512 154 / 91; 4/4 heads, 16 sequences of
// 2048: 64 rows 61 / 72, 128 113 / 77, of 32768 64 608 / 972, 128 1103 / 973; 32/8
// heads of 128, 8192 keys: 128 rows 25 / 38, 256 39 / 40, 8 sequences of 32768: 64 222
// / 472, 256 764 / 608; 14/2 heads of 64, 8192 keys: 1022 rows 26 / 33, 32768 keys:
// 511 41 / 45, 1022 70 / 50. One query position is always kvq_few's, which alone
// applies the gate.
bool kvq_is_few(long long rows, int B, int KVH, int L, int D, int C) {
  if (L == 1 || rows <= 96) return true;
  const double work = (double)rows * B * KVH * C * D, root = std::sqrt((double)C);
  return work <= 1.76e6 * root * std::sqrt(root) && work <= (D == 64 ? 3.0e9 : 4.29e9);  // C^(3/4)
}
// Rows a block of kvq_few holds: as few columns as the row count needs, as a
// block's vector work grows with its column tiles. In heads of 256 sixteen rows
// leave one wave on a SIMD, which 4-bit codes feel until the second reading of
// the keys costs more. 8 a block / 16, us, 8/2 heads of 256, 4 bits: 12 rows
// after 1024 tokens 8.9 / 11.4, after 32768 16.5 / 22.9; 64 rows 16.7 / 24.7 and
// 30 / 37, 6 sequences of 32768 124 / 127; 128 rows there 288 / 233. In 8 bits 12
// rows 10.1 / 12.3 and 26 / 26, 6 sequences 68 / 58; 64 rows 217 / 149.
int kvq_block_rows(int D, int bits, long long rows) {
  if (D == 64) return 16;
  if (D == 128) return rows <= 8 ? 8 : 16;
  return rows <= 4 ? 4 : rows <= (bits == 4 ? 64 : 8) ? 8 : 16;
}
// Workgroups of a launch of `units` KV heads x row blocks, up to which their keys
// are split: one a CU for the long rows of one block, which are bound by memory,
// and for all of 256 bytes, which leave a SIMD one wave; two a CU for shorter ones
// and several blocks, and where whole splits would leave a fifth of the CUs idle.
// 256 / 512, us, one token after 131071: 8/2 heads of 256 20.5 / 22.5 (8 bits 31.0
// / 36.9), 32/8 heads of 128 in 8 bits 47.9 / 52.2, in 4 bits 35.3 / 33.5, 14/2
// heads of 64, 8 sequences 51.4 / 40.3; 16 tokens after 32768, 6 sequences, 8/2
// heads of 256 186 / 124 (8 bits 142 / 149); 1024 was never better.
int kvq_target(int D, int bits, int blocks, long long units) {
  const int row = D * bits / 8;
  return row >= (blocks == 1 ? 128 : 256) && 256 / units * units >= 208 ? 256 : 512;
}
// Splits of every KV head's keys: from the capacity, as the valid length is not
// known here.
int kvq_splits(int B, int KVH, int blocks, int D, int bits, int C) {
  const long long pieces = (C + 127) / 128, units = (long long)B * KVH * blocks;
  long long s = kvq_target(D, bits, blocks, units) / units;
  s = s < 1 ? 1 : s > kKvqSplits ? kKvqSplits : s;
  return (int)(s < pieces ? s : pieces);
}
// How a call's row blocks spread over workgroups, and its workspace.
struct KvqFewPlan {
  int hp, blocks, splits, share;
  long long floats;
};
KvqFewPlan kvq_few_plan(int B, int KVH, long long rows, int D, int bits, int C, bool lengths) {
  KvqFewPlan p;
  p.hp = kvq_block_rows(D, bits, rows);
  p.blocks = (int)((rows + p.hp - 1) / p.hp);
  p.splits = kvq_splits(B, KVH, p.blocks, D, bits, C);
  // several sequences with lengths of their own and one block: shared
  p.share = 0;
  const long long most = (long long)((C + 127) / 128) * B;  // pieces of a KV head
  if (lengths && B > 1 && B <= kKvqShared && p.blocks == 1) {
    const int s = kvq_target(D, bits, 1, KVH) / KVH;
    p.share = s < 1 ? 1 : s > kKvqSplits ? kKvqSplits : s;
    if (p.share > most) p.share = (int)most;
  }
  const long long fixed = (long long)B * KVH * p.blocks * p.splits, shared = (long long)KVH * (p.share + B);
  p.floats = (fixed > shared ? fixed : shared) * p.hp * (D + 2);
  return p;
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
  Q35_CHECK_ARG(B < 65536 && KVH < 32768 && (long long)B * KVH < (1ll << 31));
  const KvqSrc ks{(const uint16_t*)k, k_sb, k_sh, k_sl}, vs{(const uint16_t*)v, v_sb, v_sh, v_sl};
  const dim3 grid(((unsigned)L + 15) / 16, 2 * (unsigned)KVH, (unsigned)B);
#define Q35_CALL(E, BITS)                                                                                         \
  kvq_write<E, BITS><<<grid, 256, 0, stream>>>(ks, vs, (uint8_t*)kq, (uint8_t*)vq, (uint32_t*)kp, (uint32_t*)vp,   \
                                               (const long long*)start_dev, n_start, start, KVH, L, capacity)
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
  Q35_CHECK_ARG(B < 65536 && KVH < 32768 && (long long)B * KVH < (1ll << 31));
  const dim3 grid(((unsigned)L + 15) / 16, 2 * (unsigned)KVH, (unsigned)B);
#define Q35_CALL(E, BITS)                                                                                          \
  kvq_read<E, BITS><<<grid, 256, 0, stream>>>((const uint8_t*)kq, (const uint8_t*)vq, (const uint32_t*)kp,          \
                                              (const uint32_t*)vp, (uint16_t*)k, (uint16_t*)v, start, L, KVH, capacity)
  Q35_KVQ_BY_D(Q35_CALL);
#undef Q35_CALL
  return q35_last_error();
}

long long q35_gqa_attention_kvq_workspace(int B, int QH, int KVH, int L, int D, int bits, int capacity) {
  if (!kvq_shape_ok(B, KVH, L, D, bits, capacity) || QH <= 0 || QH % KVH) return -1;
  const long long rows = (long long)(QH / KVH) * L;
  if ((long long)B * L == 0) return 0;
  if (!kvq_is_few(rows, B, KVH, L, D, capacity)) return kvq_prompt_workspace(B, QH, KVH, L, D, capacity);
  return kvq_few_plan(B, KVH, rows, D, bits, capacity, true).floats;
}

int q35_gqa_attention_kvq(const void* q, const void* kq, const void* vq, const void* kp, const void* vp,
                          const void* len_dev, int n_len, long long offset, const void* gate, long long gate_stride,
                          float scale, void* out, void* workspace, long long workspace_floats, int B, int QH, int KVH,
                          int L, int D, int bits, int capacity, hipStream_t stream) {
  Q35_CHECK_ARG(kvq_shape_ok(B, KVH, L, D, bits, capacity) && QH > 0 && QH % KVH == 0);
  if ((long long)B * L == 0) return 0;
  Q35_CHECK_ARG(!len_dev || n_len == 1 || n_len == B);
  Q35_CHECK_ARG(!gate || (L == 1 && gate_stride % 4 == 0 && gate_stride >= 0 && gate_stride < (1ll << 31)));
  Q35_CHECK_ARG(q && kq && vq && kp && vp && out && q35_aligned16(kq) && q35_aligned16(vq) && q35_aligned16(kp) &&
                q35_aligned16(vp) && q35_aligned16(q) && q35_aligned16(out) && q35_aligned8(gate));
  const long long rows = (long long)(QH / KVH) * L;
  Q35_CHECK_ARG((long long)B * KVH * rows < (1ll << 31));
  if (kvq_is_few(rows, B, KVH, L, D, capacity)) {
    const KvqFewPlan p = kvq_few_plan(B, KVH, rows, D, bits, capacity, len_dev && n_len > 1);
    Q35_CHECK_ARG(B < 65536 && KVH < 65536 && workspace && q35_aligned16(workspace) && workspace_floats >= p.floats);
    const KvqShape shape{(const long long*)len_dev, offset, n_len, KVH, L, capacity, p.blocks, p.splits, QH / KVH, B,
                         p.share};
    const KvqArgs a{shape, scale, (const uint16_t*)q, (const uint8_t*)kq, (const uint8_t*)vq, (const uint32_t*)kp,
                    (const uint32_t*)vp, (float*)workspace};
    const KvqMergeArgs m{shape, (int)gate_stride, (const float*)workspace, (const uint16_t*)gate, (uint16_t*)out};
    const long long units = (long long)B * KVH * p.splits, round = units < 8 ? units : 8;
    const long long wgs = (units + round - 1) / round * round * p.blocks;
    Q35_CHECK_ARG(wgs < (1ll << 31));
    const dim3 grid = p.share ? dim3((unsigned)((p.share + B) * KVH))
                      : p.blocks == 1 ? dim3((unsigned)p.splits, (unsigned)KVH, (unsigned)B) : dim3((unsigned)wgs);
    const int most = p.share ? p.share : p.splits, hp = p.hp;  // records of a row
    const dim3 mgrid((unsigned)(rows * (D / 64)), (unsigned)KVH, (unsigned)B);
#define Q35_FEW(DD, HP)                                                            \
  do {                                                                             \
    if (bits == 4) kvq_few<DD, 4, HP><<<grid, 256, 0, stream>>>(a);                \
    else kvq_few<DD, 8, HP><<<grid, 256, 0, stream>>>(a);                          \
    if (most <= 16) kvq_few_merge<DD, HP, 1><<<mgrid, 256, 0, stream>>>(m);      \
    else if (most <= 64) kvq_few_merge<DD, HP, 4><<<mgrid, 256, 0, stream>>>(m); \
    else kvq_few_merge<DD, HP, 16><<<mgrid, 256, 0, stream>>>(m);                  \
  } while (0)
    if (D == 64) Q35_FEW(64, 16);
    else if (D == 128 && hp == 8) Q35_FEW(128, 8);
    else if (D == 128) Q35_FEW(128, 16);
    else if (hp == 4) Q35_FEW(256, 4);
    else if (hp == 8) Q35_FEW(256, 8);
    else Q35_FEW(256, 16);
#undef Q35_FEW
    return q35_last_error();
  }
  Q35_CHECK_ARG(workspace && q35_aligned16(workspace) &&
                workspace_floats >= kvq_prompt_workspace(B, QH, KVH, L, D, capacity));
  return kvq_prompt(q, kq, vq, kp, vp, (const long long*)len_dev, n_len, offset, scale, out, (float*)workspace, B, QH,
                    KVH, L, D, bits, capacity, stream);
}

}  // extern "C"
