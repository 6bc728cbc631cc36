// What the kernels of the K/V cache in 4 or 8 bits share: its form is described in
// kvq.hip.
#pragma once
#include "q35_tile.hpp"

namespace {

Q35_DEV uint32_t kvq_code(uint32_t w, int i, int bits) { return bits == 4 ? (w >> (4 * i)) & 15u : (w >> (8 * i)) & 255u; }

// 2^e for -126 <= e <= 127; the e that brings x > 0 to [2^to, 2^(to + 1)) by 2^e (a
// bf16 x is below 2^128, and below 2^-112 it is left smaller).
Q35_DEV float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
Q35_DEV int kvq_shift(float x, int to) {
  if (!(x > 0.f)) return 0;
  const int e = to - ilogbf(x);
  return e < -120 ? -120 : e > 126 ? 126 : e;
}

typedef uint32_t q35_u32x2 __attribute__((ext_vector_type(2)));

// What the few-row kernels take, in as few bytes as it needs: a launch of 192 bytes
// of arguments takes the host 1 us longer than one of 8.
struct KvqShape {
  const long long* len;
  long long offset;
  int n_len, KVH, L, C, blocks, splits, G, B;  // G query heads a KV head
  int share;  // workgroups that a KV head's sequences share by their lengths; 0: `splits` for each
};
struct KvqArgs : KvqShape {
  float scale;
  const uint16_t* q;
  const uint8_t *kq, *vq;
  const uint32_t *kp, *vp;
  float* part;
};
struct KvqMergeArgs : KvqShape {
  int gate_stride;
  const float* part;
  const uint16_t* gate;
  uint16_t* out;
};

// Row r is head r % G of token r / G; a decoded token's rows need no division.
Q35_DEV int kvq_token(const KvqShape& a, int r) { return a.L == 1 ? 0 : (int)((unsigned)r / (unsigned)a.G); }
// Keys that token i of a sequence that starts at `start` sees.
Q35_DEV int kvq_limit(const KvqShape& a, long long start, int i) {
  const long long n = start + i + 1;
  return (int)(n < 0 ? 0 : n > a.C ? a.C : n);
}
Q35_DEV long long kvq_start(const KvqShape& a, int b) {
  return (a.len ? a.len[a.n_len > 1 ? b : 0] : 0) + a.offset;
}

// The values of run c of a row: src its codes, ps the row's first param, groups C
// apart.
template <int E, int BITS>
Q35_DEV void kvq_run(const uint8_t* src, const uint32_t* ps, int C, bool values, int c, float (&x)[E]) {
  constexpr int NG = E / 4;
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
#pragma unroll
  for (int e = 0; e < E; ++e)
    x[e] = fmaf((float)kvq_code(w[e * BITS / 32], e % (32 / BITS), BITS), bf_lo(p[e / 4]), bf_hi(p[e / 4]));
}

// ---------------------------------------------------------------- read back
// The same 16 lanes a row: bf16(fma(code, step, low)), one rounding. Bound by
// memory: 131072 tokens of 2 heads of 256 in 8 bits (411 MB) 73 us, 5.6 TB/s, where a
// large copy reaches 4.9; 777 tokens 2.5 us, a launch.
template <int E, int BITS>
__global__ __launch_bounds__(256) void kvq_read(const uint8_t* __restrict__ kq, const uint8_t* __restrict__ vq,
                                                const uint32_t* __restrict__ kp, const uint32_t* __restrict__ vp,
                                                uint16_t* __restrict__ k, uint16_t* __restrict__ v, int start,
                                                int L, int KVH, int C) {
  constexpr int NG = E / 4, RB = 2 * E * BITS;
  const unsigned t = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (t >= (unsigned)L) return;
  const int c = threadIdx.x & 15;
  const unsigned bh = blockIdx.z * KVH + (blockIdx.y >> 1), pos = start + t;
  const bool values = blockIdx.y & 1;
  const uint8_t* src = (values ? vq : kq) + ((size_t)bh * C + pos) * RB + c * (E * BITS / 8);
  const uint32_t* ps = (values ? vp : kp) + (size_t)bh * NG * C + pos;
  float x[E];
  kvq_run<E, BITS>(src, ps, C, values, c, x);
  uint32_t o[E / 2];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) o[e] = pack_bf2(x[2 * e], x[2 * e + 1]);
  uint16_t* dst = (values ? v : k) + ((size_t)bh * L + t) * (16 * E) + E * c;
  if constexpr (E == 4) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
  } else {
#pragma unroll
    for (int j = 0; j < E / 8; ++j)
      *reinterpret_cast<uint4*>(dst + 8 * j) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
  }
}

}  // namespace

// Attention of many query rows (kvq_prompt.hip): workspace floats and launch.
long long kvq_prompt_workspace(int B, int QH, int KVH, int L, int D, int C);
int kvq_prompt(const void* q, const void* kq, const void* vq, const void* kp, const void* vp, const long long* len,
               int n_len, long long offset, float scale, void* out, float* workspace, int B, int QH, int KVH, int L,
               int D, int bits, int C, hipStream_t stream);
