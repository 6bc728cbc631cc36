// Causal GQA attention of many query rows over the K/V cache in 4 or 8 bits: the
// cache's values in a workspace, unpacked once, and flash attention on the matrix
// cores over those.
//
// A row tile of 128 rows reads every key once, so a prompt of n rows would
// unpack a cache n / 128 times inside the attention; unpacked once, its blocks
// go from memory straight into LDS. 4096 tokens after 28000 (8/2 heads of 256, 8
// bits) take 947 to 970 us, 27 of them unpacking and 13 the merge of two ranges:
// 1040 TFLOP/s and more in all, where a large library product reaches 1384.
//
// The values are held in 16 bits as fp16 times one power of two per head that
// brings the greatest of them (by the params, over the keys that are seen) to
// 2^14: 11 significant bits down to 2^-28 of it, 2^-12 off at most (bf16 would be
// 2^-8, more than an 8-bit cache's own step). Queries are exact in fp16 times a
// power of two of their row, but for values below 2^-21 of its greatest.
#include "kvq.hpp"

namespace {

Q35_DEV uint2 lds_read_tr16(const void* p) {
  typedef short q35_i16x4 __attribute__((ext_vector_type(4)));
  const q35_i16x4 v =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) q35_i16x4*)(p));
  return __builtin_bit_cast(uint2, v);
}

constexpr int kFaKeys = 64;       // keys per block
constexpr int kFaWaves = 4;
constexpr int kFaRows = 32 * kFaWaves;  // query rows per tile
constexpr int kFaMaxSplits = 64;
constexpr int kFaRanges = 64;     // partial maxima of a head's keys or values
// Up to this capacity every unpacking workgroup finds the maximum itself; above,
// a launch of its own finds partial maxima. Self / launch, us, 8/2 heads of 256: 1000
// tokens of 1024 33.1 / 35.1, 300 of 2048 38.4 / 38.9, 1000 of 4096 63.9 / 61.8, 300
// of 8192 64.2 / 57.7.
constexpr int kFaSelf = 2048;

typedef _Float16 q35_f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 q35_f16x8 __attribute__((ext_vector_type(8)));
Q35_DEV uint32_t pack_h2(float lo, float hi) {
  const q35_f32x2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, q35_f16x2));
}
Q35_DEV q35_f32x16 mfma32h(const q35_u32x4 a, const q35_u32x4 b, q35_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(q35_f16x8, a), __builtin_bit_cast(q35_f16x8, b), c,
                                                0, 0, 0);
}
struct UnpackArgs {
  const uint8_t *kq, *vq;
  const uint32_t *kp, *vp;
  const long long* len;
  int n_len;
  long long offset;  // of the last token: it sees positions up to len + offset
  uint16_t *k, *v;
  float *ranges, *scales;  // [B * KVH, 2, kFaRanges], [B * KVH, 2]
  int* flags;              // [B * KVH, C / 64 rounded up]: whether a block of values holds an infinity or NaN
  int KVH, n, C;
};
// Rows of a head that are seen.
Q35_DEV int unpack_rows(const UnpackArgs& a, int bh) {
  if (!a.len) return a.n;
  const long long last = a.len[a.n_len > 1 ? bh / a.KVH : 0] + a.offset;
  return (int)(last < 0 ? 0 : last >= a.n ? a.n : last + 1);
}
// The greatest finite magnitude of the groups that thread t of `threads` takes
// of a head's first n rows.
template <int NG, int BITS>
Q35_DEV float fa_greatest(const uint32_t* p, int n, int C, int t, int threads) {
  constexpr float T = BITS == 4 ? 15.f : 255.f;
  float m = 0.f;
  for (int i = 4 * t; i < n; i += 4 * threads) {
    uint4 x[NG];  // requested together: group by group was one memory round trip each
#pragma unroll
    for (int g = 0; g < NG; ++g) x[g] = *reinterpret_cast<const uint4*>(p + (size_t)g * C + i);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint32_t w[4] = {x[g].x, x[g].y, x[g].z, x[g].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = fmaxf(fabsf(bf_hi(w[e])), fabsf(fmaf(T, bf_lo(w[e]), bf_hi(w[e]))));
        if (i + e < n && y < INFINITY) m = fmaxf(m, y);
      }
    }
  }
  return m;
}
Q35_DEV float fa_block_max(float m, float* red) {  // of 256 threads
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// Partial maxima of long caches, grid (kFaRanges, keys and values, heads).
template <int NG, int BITS>
__global__ __launch_bounds__(256) void kvq_ranges(const UnpackArgs a) {
  __shared__ float red[4];
  const int bh = blockIdx.z;
  const uint32_t* p = (blockIdx.y ? a.vp : a.kp) + (size_t)bh * NG * a.C;
  const float m = fa_block_max(
      fa_greatest<NG, BITS>(p, unpack_rows(a, bh), a.C, blockIdx.x * 256 + threadIdx.x, 256 * kFaRanges), red);
  if (threadIdx.x == 0) a.ranges[(bh * 2 + blockIdx.y) * kFaRanges + blockIdx.x] = m;
}

// 64 rows a workgroup, 16 lanes a row; grid (blocks, keys and values, heads). Bound
// by memory in a long cache, by two round trips (params, rows) in a short one: 1024
// positions of 2 heads of 256 take 6.7 us.
template <int E, int BITS>
__global__ __launch_bounds__(256) void kvq_unpack(const UnpackArgs a) {
  constexpr int NG = E / 4, RB = 2 * E * BITS;
  __shared__ float red[4];
  const int bh = blockIdx.z, n = unpack_rows(a, bh), values = blockIdx.y, t = threadIdx.x, c = t & 15;
  if (blockIdx.x > 0 && (int)blockIdx.x * kFaKeys >= n) return;
  const uint32_t* p = (values ? a.vp : a.kp) + (size_t)bh * NG * a.C;
  const uint8_t* src = (values ? a.vq : a.kq) + (size_t)bh * a.C * RB + c * (E * BITS / 8);
  uint16_t* dst = (values ? a.v : a.k) + (size_t)bh * a.C * (16 * E) + E * c;
  // the workgroup's rows, requested before the maximum is known
  const int r0 = blockIdx.x * kFaKeys + (t >> 4);
  float x[kFaKeys / 16][E];
#pragma unroll
  for (int j = 0; j < kFaKeys / 16; ++j) {
    const int r = min(r0 + 16 * j, max(n, 1) - 1);
    kvq_run<E, BITS>(src + (size_t)r * RB, p + r, a.C, values, c, x[j]);
  }
  float m;
  if (a.ranges) {
    m = t < kFaRanges ? a.ranges[(bh * 2 + values) * kFaRanges + t] : 0.f;
  } else {
    m = fa_greatest<NG, BITS>(p, n, a.C, t, 256);
  }
  const int shift = kvq_shift(fa_block_max(m, red), 14);
  const float up = exp2_int(shift);
  if (values) {
    float z = 0.f;  // NaN if any value is not finite
#pragma unroll
    for (int j = 0; j < kFaKeys / 16; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) z += x[j][e] * 0.f;
    const bool bad = __syncthreads_or(z != z);
    if (t == 0) a.flags[(size_t)bh * ((a.C + kFaKeys - 1) / kFaKeys) + blockIdx.x] = bad;
  }
  if (blockIdx.x == 0 && t == 0) a.scales[bh * 2 + values] = exp2_int(-shift);
#pragma unroll
  for (int j = 0; j < kFaKeys / 16; ++j) {
    const int r = r0 + 16 * j;
    if (r >= n) return;
    uint32_t o[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) o[e] = pack_h2(x[j][2 * e] * up, x[j][2 * e + 1] * up);
    uint16_t* d = dst + (size_t)r * (16 * E);
    if constexpr (E == 4) {
      *reinterpret_cast<uint2*>(d) = make_uint2(o[0], o[1]);
    } else {
#pragma unroll
      for (int i = 0; i < E / 8; ++i)
        *reinterpret_cast<uint4*>(d + 8 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    }
  }
}

template <int D>
struct FaShape {
  static constexpr int ROW = 2 * D;                  // bytes of a K or V row
  static constexpr int BLOCK = kFaKeys * ROW;        // of a block
  static constexpr int CPR = ROW / 16;               // 16-byte chunks of a row
  static constexpr int NC = BLOCK / 1024 / kFaWaves; // a wave's copies of a block
  static constexpr int KS = D / 16, ND = D / 32;     // k steps of S, dim tiles of O
  static constexpr int REC = 16 * D + 64;            // floats of a wave's split record: O / l as fp16, (m, l)
  static constexpr int WAVES = D > 64 ? 1 : 2;     // waves a SIMD
};

// 16-byte chunk c of a staged row r sits at slot c ^ fa_swz(r): the 16 rows of a
// K fragment read and the 4 rows x 4 chunks of a transposed V read each fall on
// 16 distinct bank groups.
template <int D>
Q35_DEV uint32_t fa_swz(uint32_t r) {
  if (D == 64) {
    const uint32_t x = r >> 1 & 7;
    return ((x & 1) << 2) | (x >> 1);
  }
  return ((r & 3) << 2) | ((r >> 2) & 3);
}

struct FaArgs {
  const uint16_t *q, *K, *V;  // K, V [B * KVH, C, D] fp16
  const float* scales;        // [B * KVH, 2]: the values are these times them
  const int* flags;           // [B * KVH, blocks]: V has infinities or NaN
  const long long* len;
  int n_len;
  long long offset;
  float scale;
  uint16_t* out;
  float* part;
  int QH, KVH, L, C, G, R, tiles, splits, bhs;
};
Q35_DEV long long fa_start(const FaArgs& a, int b) { return (a.len ? a.len[a.n_len > 1 ? b : 0] : 0) + a.offset; }
// Keys that row r sees.
Q35_DEV int fa_limit(const FaArgs& a, long long start, int r) {
  const long long n = start + (int)((unsigned)r / (unsigned)a.G) + 1;
  return (int)(n < 0 ? 0 : n > a.C ? a.C : n);
}
// Key blocks per range of a tile with nblk of them: over at most `splits`
// ranges, of at least two blocks.
Q35_DEV int fa_range(const FaArgs& a, int nblk) { return max((nblk + a.splits - 1) / a.splits, min(nblk, 2)); }

// ------------------------------------------------- attention of many rows
// Products are transposed: a wave owns 32 query rows (row = token x head of one
// KV head, so any head grouping fills its tiles) as the COLUMNS of every
// v_mfma_f32_32x32x16_f16,
//   S^T = K Q^T  (A = 32 keys x 16 dims from LDS, B = Q^T held in registers),
//   O^T += V^T P^T  (A = 32 dims x 16 keys from LDS, B = P^T),
// so a lane holds one query row: the softmax needs no cross-lane step but one
// exchange between lanes l and l ^ 32 per block, and the C layout of S^T is,
// with the 16 keys of a k step taken in the order {0-3, 8-11 | 4-7, 12-15},
// already the B operand of O^T: P, rounded to fp16, never leaves the registers.
// V rows reach the A operand through the transpose read ds_read_b64_tr_b16:
// within a 16-lane group, lane 4 e + q points at row e, column 4 q and lane i
// receives the 4 rows of column i.
//
// The 4 waves of a workgroup are 4 tiles of 32 rows that share the K and V
// blocks in LDS (two buffers each, rows copied straight into LDS a whole block
// ahead, one barrier per block). Vector work is interleaved by hand: the MFMAs
// of S for block j + 1 carry the copies of the following blocks and half of the
// exponentials of block j, the MFMAs of O the other half, the packing of P and
// the scale and row maximum of block j + 1.
//
// Bound by the matrix cores and the power they draw: 128 KB of LDS leave one
// workgroup a CU in heads of 256, a block takes 2.1 us where its products alone are
// 0.9 at the full clock. A short prompt is bound by latency: of 1000 tokens' 18 us,
// 5 pass until the first block and Q are there and 2.4 with each of up to 4 blocks.
//
// The running maximum m (in units of log2) moves only when a row's block maximum
// passes it by 8, so O is rescaled a few times per row; P is 2^(s - m + 7), below
// 2^15, with 11 bits down to 2^-21 of the weight at m.
//
// Keys past a tile's last one are clamped to it on load and, like every key
// past a row's own end, masked to -inf in S. In blocks where some row's end
// lies, V's infinities and NaN (the unpacking flags their blocks) are taken out
// and their dims set to NaN at the end for the rows that see them: a weight of
// zero would not hide them.
template <int D>
__global__ __launch_bounds__(kFaWaves * 64, (FaShape<D>::WAVES)) void kvq_fa(const FaArgs a) {
  using F = FaShape<D>;
  constexpr int KS = F::KS, ND = F::ND, NC = F::NC, ROW = F::ROW, BLOCK = F::BLOCK;
  constexpr int LA = 3;  // K fragments read ahead
  // K buffers at 0 and BLOCK, V buffers at 2 and 3 BLOCK
  __shared__ alignas(1024) uint8_t lds[4 * BLOCK];
  __shared__ int bad_s[D];  // first key of a masked block with a dim's V not finite
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int l32 = lane & 31, kh = lane >> 5;
  // The last split of every tile, late tiles first, down to split 0, which is
  // the rest: the longest ranges start first.
  const int bh = (int)(blockIdx.x % (unsigned)a.bhs), at = (int)(blockIdx.x / (unsigned)a.bhs);
  const int tile = a.tiles - 1 - at % a.tiles, split = a.splits - 1 - at / a.tiles;
  const int b = bh / a.KVH, kvh = bh % a.KVH;
  const int r0 = tile * kFaRows, rw = r0 + 32 * w;
  const long long start = fa_start(a, b);
  const int n_keys = fa_limit(a, start, min(r0 + kFaRows, a.R) - 1);
  const int nblk = (n_keys + kFaKeys - 1) / kFaKeys;
  const int sb = fa_range(a, nblk), nsplit = nblk ? (nblk + sb - 1) / sb : 1;
  if (split >= nsplit) return;  // whole workgroup: no barrier is skipped
  const int row = min(rw + l32, a.R - 1);
  const int tok = (int)((unsigned)row / (unsigned)a.G), head = kvh * a.G + (row - tok * a.G);
  uint16_t* orow = a.out + (((size_t)b * a.L + tok) * a.QH + head) * D;
  if (nblk == 0) {  // no row of the tile sees a key
    if (rw + l32 < a.R)
      for (int d = 8 * kh; d < D; d += 16) *reinterpret_cast<uint4*>(orow + d) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int b1 = nblk - (nsplit - 1 - split) * sb, b0 = split ? b1 - sb : 0;
  const uint8_t* Kh = (const uint8_t*)(a.K + (size_t)bh * a.C * D);
  const uint8_t* Vh = (const uint8_t*)(a.V + (size_t)bh * a.C * D);

  // ---- copies: wave w takes 1 KiB pieces w + 4 i of each block
  const uint32_t cr = (1024u / ROW) * w + lane / F::CPR, cstep = 4u * (1024u / ROW);  // row of copy i: cr + cstep i
  const uint32_t cc[2] = {16u * ((uint32_t)(lane % F::CPR) ^ fa_swz<D>(cr)),
                          16u * ((uint32_t)(lane % F::CPR) ^ fa_swz<D>(cr + cstep))};
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_offset(lds) + 1024u * (uint32_t)w);
  auto copy = [&](const uint8_t* base, uint32_t to, int blk, int i) {
    const uint32_t r = min(cr + cstep * i, (uint32_t)(n_keys - 1 - blk * kFaKeys));
    dma16(lds0 + to + 4096u * i, base + (size_t)blk * BLOCK, r * ROW + cc[i & 1]);
  };

  // K and V of the first block and K of the second, ahead of Q's preparation
#pragma unroll
  for (int i = 0; i < NC; ++i) copy(Kh, 0, b0, i);
#pragma unroll
  for (int i = 0; i < NC; ++i) copy(Vh, 2u * BLOCK, b0, i);
#pragma unroll
  for (int i = 0; i < NC; ++i) copy(Kh, BLOCK, min(b0 + 1, b1 - 1), i);

  // ---- fragment addresses; the buffer is added by ^ BLOCK
  // K: row l32 of a 32-key half (the second half BLOCK / 2 on), chunk 2 s + kh
  uint32_t ka[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) ka[s] = (uint32_t)l32 * ROW + 16u * ((2u * s + kh) ^ fa_swz<D>(l32));
  // V: rows 4 kh + e and 4 kh + 8 + e of a 16-key step, dims 32 d + 16 ((lane /
  // 16) % 2) + 4 (lane % 4)
  uint32_t va[2][ND];
  {
    const uint32_t e = (lane & 15) >> 2, cl = 2u * ((lane >> 4) & 1) + ((lane >> 1) & 1);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t r = 4u * kh + 8u * u + e;
#pragma unroll
      for (int d = 0; d < ND; ++d)
        va[u][d] = 2u * BLOCK + r * ROW + 16u * ((4u * d + cl) ^ fa_swz<D>(r)) + 8u * (lane & 1);
    }
  }

  // ---- Q: column l32 of the B operand, dims 16 s + 8 kh .., in fp16 with the
  // row's greatest brought to [2^14, 2^15)
  q35_u32x4 qf[KS];
  float c2 = a.scale * 1.4426950408889634f * a.scales[2 * bh];
  {
    const uint16_t* qp = a.q + (((size_t)b * a.QH + head) * a.L + tok) * D + 8 * kh;
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[s] = *reinterpret_cast<const q35_u32x4*>(qp + 16 * s);
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(fabsf(bf_lo(qf[s][e])), fabsf(bf_hi(qf[s][e]))));
    }
    const int shift = kvq_shift(half_max(top), 14);
    const float up = exp2_int(shift);
    c2 *= exp2_int(-shift);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[s][e] = pack_h2(bf_lo(qf[s][e]) * up, bf_hi(qf[s][e]) * up);
  }
  // Q stays in AGPRs, which the MFMAs read as they are
  if constexpr (D == 256) {
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+a"(qf[s]));
  }
  const int limit = fa_limit(a, start, row);
  const int least = fa_limit(a, start, min(rw, a.R - 1));     // of the wave's rows
  const int least_wg = fa_limit(a, start, r0);                // of the workgroup's
  const int* flags = a.flags + (size_t)bh * ((a.C + kFaKeys - 1) / kFaKeys);
  bool bad = false;

  q35_f32x16 o[ND], sc[2], sn[2];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = -INFINITY, l = 0.f, mx = -INFINITY;

  // ---- S of the first block
  wait_vm<0>();
  __syncthreads();
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) sn[t][r] = 0.f;
#pragma unroll
  for (int x = 0; x < 2 * KS; ++x)
    sn[x & 1] = mfma32h(*reinterpret_cast<const q35_u32x4*>(lds + ka[x >> 1] + (BLOCK / 2) * (x & 1)), qf[x >> 1], sn[x & 1]);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      sc[t][r] = sn[t][r] * c2;
      mx = fmaxf(mx, sc[t][r]);
    }
#pragma unroll
  for (int s = 0; s < KS; ++s) ka[s] ^= (uint32_t)BLOCK;
  __syncthreads();  // the loop's first copies go where this K was

  // ---- one block: sc holds its scaled scores, mx their maximum over the
  // lane's keys; ka points at K of the next block, va at V of this one. The last
  // block computes the scores of itself again in place of a next one's: a form
  // of its own would double the code, which a short range reads cold.
  for (int blk = b0; blk < b1; ++blk) {
    const uint32_t kbuf = (blk - b0) & 1 ? BLOCK : 0;  // free: this block's K, the last one's V
    const uint32_t vbuf = 2u * BLOCK + (BLOCK - kbuf);
    if (blk * kFaKeys + kFaKeys > least_wg && flags[blk]) {  // uniform over the workgroup
      uint8_t* vb = lds + 2 * BLOCK + kbuf;
      if (!bad)
        for (int d = threadIdx.x; d < D; d += 256) bad_s[d] = 0x7fffffff;
      bad = true;
      __syncthreads();
      for (int i = threadIdx.x; i < BLOCK / 2; i += 256) {
        const int r = i / D, d = i % D;
        uint16_t* p = (uint16_t*)(vb + r * ROW + 16 * ((uint32_t)(d / 8) ^ fa_swz<D>(r)) + 2 * (d % 8));
        if ((*p & 0x7c00) == 0x7c00) {
          *p = 0;
          atomicMin(&bad_s[d], blk * kFaKeys + r);
        }
      }
      __syncthreads();
    }
    // O stays in AGPRs up to the rescale: without this the rescale's copies
    // out of them were made for every block, rescaled or not
#pragma unroll
    for (int d = 0; d < ND; ++d) asm volatile("" : "+a"(o[d]));
    q35_u32x4 kf[LA + 1], vf[2][ND], ph[2];
    auto readk = [&](int x) {
      kf[x % (LA + 1)] = *reinterpret_cast<const q35_u32x4*>(lds + ka[x >> 1] + (BLOCK / 2) * (x & 1));
    };
#pragma unroll
    for (int x = 0; x < LA; ++x) readk(x);
    Q35_PIN();
    if (blk * kFaKeys + kFaKeys > least) {
      mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = blk * kFaKeys + 32 * t + 8 * (r >> 2) + 4 * kh + (r & 3);
          if (key >= limit) sc[t][r] = -INFINITY;
          mx = fmaxf(mx, sc[t][r]);
        }
    }
    mx = half_max(mx);
    if (__ballot(mx > m + 8.f)) {
#pragma unroll
      for (int d = 0; d < ND; ++d) asm volatile("" : "+a"(o[d]));
      const float mn = fmaxf(m, mx);
      const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= corr;
      if (__ballot(m != -INFINITY)) {  // else O is still zero
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= corr;
#pragma unroll
        for (int d = 0; d < ND; ++d) asm volatile("" : "+a"(o[d]));
      }
      m = mn;
    }
    // A row without any key so far keeps m = -inf: subtract 0 then.
    const float ms = m == -INFINITY ? 0.f : m - 7.f;

    float l1 = 0.f;
    auto ex = [&](int z) {  // exponential of element z
      const float p = __builtin_amdgcn_exp2f(sc[z >> 4][z & 15] - ms);
      sc[z >> 4][z & 15] = p;
      if (z & 1) l1 += p;
      else l += p;
    };
    auto pack = [&](int kk, int e) {  // P of elements 2 e, 2 e + 1 of k step kk
      ph[kk & 1][e] = pack_h2(sc[kk >> 1][8 * (kk & 1) + 2 * e], sc[kk >> 1][8 * (kk & 1) + 2 * e + 1]);
    };
    auto readv = [&](int kk, int d) {
      const uint2 x = lds_read_tr16(lds + va[0][d] + 16 * ROW * kk), y = lds_read_tr16(lds + va[1][d] + 16 * ROW * kk);
      vf[kk & 1][d] = q35_u32x4{x.x, x.y, y.x, y.y};
    };
    constexpr int NS = 2 * KS, EX0 = NS >= 32 ? 12 : 0, PER = NS >= 16 ? 1 : 2;
#pragma unroll
    for (int x = 0; x < NS; ++x) {
      if (x < 2) {
        q35_f32x16 zero;
#pragma unroll
        for (int r = 0; r < 16; ++r) zero[r] = 0.f;
        sn[x] = mfma32h(kf[x], qf[0], zero);
      } else {
        sn[x & 1] = mfma32h(kf[x % (LA + 1)], qf[x >> 1], sn[x & 1]);
      }
      if (x + LA < NS) readk(x + LA);
      // every other slot: the texture unit takes a 1 KiB copy in 16 cycles
      if ((x & 1) == 0 && x < 2 * NC) copy(Kh, kbuf, min(blk + 2, b1 - 1), x >> 1);
      else if ((x & 1) == 0 && x < 4 * NC) copy(Vh, vbuf, min(blk + 1, b1 - 1), (x >> 1) - NC);
#pragma unroll
      for (int z = PER * (x - EX0); z < PER * (x - EX0 + 1); ++z)
        if (z >= 0 && z < 16) ex(z);
      if (x >= NS - ND) readv(0, x - (NS - ND));
      if (NS >= 32 && x >= NS - 4) pack(0, x - (NS - 4));
      Q35_PIN();
    }
    if constexpr (NS < 32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) pack(0, e);
    }
    mx = -INFINITY;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
      for (int y = 0; y < ND; ++y) {
        o[y] = mfma32h(vf[kk & 1][y], ph[kk & 1], o[y]);
        if (kk < 3) {
          readv(kk + 1, y);
          if (kk < 2) {
#pragma unroll
            for (int z = 8 * y / ND; z < 8 * (y + 1) / ND; ++z) ex(16 + 8 * kk + z);
          }
#pragma unroll
          for (int e = 4 * y / ND; e < 4 * (y + 1) / ND; ++e) pack(kk + 1, e);
        }
        if (kk >= 2) {
#pragma unroll
          for (int z = 16 * (kk - 2) + 16 * y / ND; z < 16 * (kk - 2) + 16 * (y + 1) / ND; ++z) {
            const float t = sn[z >> 4][z & 15] * c2;  // into the half of sc that P no longer needs
            sc[z >> 4][z & 15] = t;
            mx = fmaxf(mx, t);
          }
        }
        Q35_PIN();
      }
    }
    l += l1;
#pragma unroll
    for (int s = 0; s < KS; ++s) ka[s] ^= (uint32_t)BLOCK;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int d = 0; d < ND; ++d) va[u][d] ^= (uint32_t)BLOCK;
    wait_vm<0>();
    __syncthreads();
  }

  l = half_sum(l);
  if (bad) {  // dims 32 d + 8 u + 4 kh + e of the lane's row
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (bad_s[32 * d + 8 * (r >> 2) + 4 * kh + (r & 3)] < limit) o[d][r] = __builtin_nanf("");
  }
  if (nsplit > 1) {
    // This split's record: O / l as fp16 (at most the greatest value, 2^15), in
    // register order (pair of quads u, u + 1 of dim tile d: 64 lanes x 16
    // bytes), then (m, l) per row. Halves in place of floats: the records of a
    // short prompt are most of its traffic.
    float* rec = a.part + ((((size_t)bh * a.tiles + tile) * a.splits + split) * kFaWaves + w) * F::REC;
    const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint4 v;
        v.x = pack_h2(o[d][8 * u] * inv, o[d][8 * u + 1] * inv);
        v.y = pack_h2(o[d][8 * u + 2] * inv, o[d][8 * u + 3] * inv);
        v.z = pack_h2(o[d][8 * u + 4] * inv, o[d][8 * u + 5] * inv);
        v.w = pack_h2(o[d][8 * u + 6] * inv, o[d][8 * u + 7] * inv);
        *reinterpret_cast<uint4*>(rec + ((d * 2 + u) * 64 + lane) * 4) = v;
      }
    if (kh == 0) *reinterpret_cast<float2*>(rec + 16 * D + 2 * l32) = make_float2(m, l);
    return;
  }
  const float inv = limit ? a.scales[2 * bh + 1] / l : 0.f;  // a row without keys is zero
  if (rw + l32 < a.R) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<uint2*>(orow + 32 * d + 8 * u + 4 * kh) =
            make_uint2(pack_bf2(o[d][4 * u] * inv, o[d][4 * u + 1] * inv),
                       pack_bf2(o[d][4 * u + 2] * inv, o[d][4 * u + 3] * inv));
  }
}

// Merge of the split records of the tiles with more than one: one workgroup per
// wave record (32 rows), O = sum_s (O / l)_s f_s / sum_s f_s, f_s = l_s 2^{m_s -
// M}, M = max_s m_s. Thread (lane, wave) adds pairs of quads in the records' own
// order.
template <int D>
__global__ __launch_bounds__(256) void kvq_fa_merge(const FaArgs a) {
  using F = FaShape<D>;
  constexpr int PER = D / 64;  // pairs of quads of a thread
  __shared__ float f_s[kFaMaxSplits][32], inv_s[32];
  const int t = threadIdx.x, lane = t & 63;
  const int w = blockIdx.x & (kFaWaves - 1), tile = blockIdx.x / kFaWaves, bh = blockIdx.y;
  const int b = bh / a.KVH, kvh = bh % a.KVH;
  const int r0 = tile * kFaRows, rw = r0 + 32 * w;
  const long long start = fa_start(a, b);
  const int n_keys = fa_limit(a, start, min(r0 + kFaRows, a.R) - 1);
  const int nblk = (n_keys + kFaKeys - 1) / kFaKeys;
  if (nblk == 0 || rw >= a.R) return;  // whole workgroup
  const int sb = fa_range(a, nblk), nsplit = (nblk + sb - 1) / sb;
  if (nsplit <= 1) return;
  const size_t rs = (size_t)kFaWaves * F::REC;
  const float* rec0 = a.part + (((size_t)bh * a.tiles + tile) * a.splits * kFaWaves + w) * F::REC;
  // (m, l) of every split and row
  __shared__ float2 ml_s[kFaMaxSplits][32];
  for (int i = t; i < 32 * nsplit; i += 256)
    ml_s[i >> 5][i & 31] = *reinterpret_cast<const float2*>(rec0 + (i >> 5) * rs + 16 * D + 2 * (i & 31));
  __syncthreads();
  if (t < 32) {
    float mx = -INFINITY, lt = 0.f;
    for (int s = 0; s < nsplit; ++s) mx = fmaxf(mx, ml_s[s][t].x);
    const float ms = mx == -INFINITY ? 0.f : mx;
    for (int s = 0; s < nsplit; ++s) {
      const float f = ml_s[s][t].y * __builtin_amdgcn_exp2f(ml_s[s][t].x - ms);  // 0 where the row saw no key
      f_s[s][t] = f;
      lt += f;
    }
    inv_s[t] = fa_limit(a, start, min(rw + t, a.R - 1)) ? a.scales[2 * bh + 1] / lt : 0.f;
  }
  __syncthreads();
  const int l32 = lane & 31, kh = lane >> 5;
  float acc[PER][8];
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[i][e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < nsplit; ++s) {
    const float f = f_s[s][l32];
    const float* rec = rec0 + s * rs + ((size_t)(t >> 6) * PER * 64 + lane) * 4;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const q35_f16x8 x = __builtin_bit_cast(q35_f16x8, *reinterpret_cast<const uint4*>(rec + i * 256));
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[i][e] = fmaf((float)x[e], f, acc[i][e]);
    }
  }
  const int row = rw + l32;
  if (row >= a.R) return;
  const float inv = inv_s[l32];
  const int tok = (int)((unsigned)row / (unsigned)a.G), head = kvh * a.G + (row - tok * a.G);
  uint16_t* orow = a.out + (((size_t)b * a.L + tok) * a.QH + head) * D + 4 * kh;
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int u = 0; u < 2; ++u)  // quad q: dims 8 q + 4 kh ..
      *reinterpret_cast<uint2*>(orow + 8 * (2 * ((t >> 6) * PER + i) + u)) =
          make_uint2(pack_bf2(acc[i][4 * u] * inv, acc[i][4 * u + 1] * inv),
                     pack_bf2(acc[i][4 * u + 2] * inv, acc[i][4 * u + 3] * inv));
}

struct FaPlan {
  int tiles, splits;
  long long part, kv, scales;  // floats of the records, of K or V, of the scales, partial maxima and flags
};
// Ranges of a tile's keys, at least two blocks each: the count with the least
// estimate, in blocks of one workgroup (2.1 us in heads of 256), of
//   the rounds of workgroups (one a CU, two in heads of 64) x the blocks of each, or
//   the longest tile's; as the capacity is full, tiles of `avg` blocks in the mean
//   + 3 blocks a round until the first is there (6 of the smaller heads' blocks)
//   + the merge, by its records.
// More tiles than a round holds are not split where most are of unequal lengths:
// the longest start first, and splits gained nothing (6000 tokens of 8/2 heads of
// 256, 376 tiles, one range 194 us, two 196). Fewer and more ranges, us: 1024 tokens
// of 8/2 heads of 256 (64 tiles) two 37.0, four 33.1, eight 41.4; 3000 tokens (188)
// one 101, two 75; 4096 (256) one 132, two 109, four 128; 748 tokens after 21874, 2
// sequences of 12/1 heads (142) two 646, seven 464; 32/8 heads of 128, 1024 tokens (256)
// one 32.6, two 38.9, 1200 after 15184 (304) one 566, three 425; 14/2 heads of 64, 1500
// tokens (166) one 30.4, three 26.0.
FaPlan fa_plan(int B, int QH, int KVH, int L, int D, int C) {
  FaPlan p;
  const long long rows = (long long)(QH / KVH) * L;
  p.tiles = (int)((rows + kFaRows - 1) / kFaRows);
  const long long wgs = (long long)p.tiles * B * KVH, nblk = (C + kFaKeys - 1) / kFaKeys;
  const long long slots = D == 64 ? 512 : 256;
  const double avg = nblk - (double)(L < C ? L : C) / (2 * kFaKeys), start = D == 256 ? 3 : 6;
  long long s = 1;
  if (wgs <= slots || avg >= 0.75 * nblk) {
    double least = 0;
    for (long long n = 1; n <= kFaMaxSplits && n <= (nblk + 1) / 2 && (n == 1 || n * wgs <= 4 * slots); ++n) {
      const double rounds = (double)((n * wgs + slots - 1) / slots), work = rounds * avg;
      const double t = (work > nblk ? work : (double)nblk) / n + start * rounds + (n > 1 ? start / 3 + n * wgs / 96.0 : 0);
      if (n == 1 || t < least) {
        least = t;
        s = n;
      }
    }
  }
  p.splits = (int)s;
  p.part = p.splits > 1 ? wgs * p.splits * kFaWaves * (16 * D + 64) : 0;
  p.kv = (long long)B * KVH * C * D / 2;
  p.scales = ((long long)B * KVH * (2 + (C > kFaSelf ? 2 * kFaRanges : 0) + nblk) + 3) / 4 * 4;
  return p;
}

}  // namespace

long long kvq_prompt_workspace(int B, int QH, int KVH, int L, int D, int C) {
  const FaPlan p = fa_plan(B, QH, KVH, L, D, C);
  return 2 * p.kv + p.part + p.scales;
}

int kvq_prompt(const void* q, const void* kq, const void* vq, const void* kp, const void* vp, const long long* len,
               int n_len, long long offset, float scale, void* out, float* workspace, int B, int QH, int KVH, int L,
               int D, int bits, int C, hipStream_t stream) {
  const FaPlan p = fa_plan(B, QH, KVH, L, D, C);
  uint16_t *K = (uint16_t*)workspace, *V = (uint16_t*)(workspace + p.kv);
  float* part = workspace + 2 * p.kv;
  float* scales = part + p.part;
  const long long bhs = (long long)B * KVH, wgs = bhs * p.tiles * p.splits;
  float* ranges = scales + 2 * bhs;
  int* flags = (int*)(ranges + (C > kFaSelf ? 2 * kFaRanges * bhs : 0));
  Q35_CHECK_ARG(wgs < (1ll << 31) && bhs < 65536);
  Q35_CHECK_ARG(len || (offset >= 0 && offset + L <= C));
  // the rows that any token may see; with the lengths on the device, those it does
  const int n = len ? C : (int)(offset + L);
  const UnpackArgs u{(const uint8_t*)kq, (const uint8_t*)vq, (const uint32_t*)kp, (const uint32_t*)vp, len, n_len,
                     offset + L - 1, K, V, C > kFaSelf ? ranges : nullptr, scales, flags, KVH, n, C};
  const dim3 ugrid((unsigned)((n + kFaKeys - 1) / kFaKeys), 2, (unsigned)bhs);
#define Q35_UNPACK(E, BITS)                                                                        \
  do {                                                                                             \
    if (u.ranges) kvq_ranges<E / 4, BITS><<<dim3(kFaRanges, 2, (unsigned)bhs), 256, 0, stream>>>(u); \
    kvq_unpack<E, BITS><<<ugrid, 256, 0, stream>>>(u);                                             \
  } while (0)
  if (bits == 4) {
    if (D == 256) Q35_UNPACK(16, 4); else if (D == 128) Q35_UNPACK(8, 4); else Q35_UNPACK(4, 4);
  } else {
    if (D == 256) Q35_UNPACK(16, 8); else if (D == 128) Q35_UNPACK(8, 8); else Q35_UNPACK(4, 8);
  }
#undef Q35_UNPACK
  const FaArgs a{(const uint16_t*)q, K, V, scales, flags, len, n_len, offset, scale, (uint16_t*)out, part, QH, KVH, L,
                 C, QH / KVH, QH / KVH * L, p.tiles, p.splits, (int)bhs};
  const dim3 mgrid((unsigned)(p.tiles * kFaWaves), (unsigned)bhs);
#define Q35_FA(DD)                                                              \
  do {                                                                          \
    kvq_fa<DD><<<(unsigned)wgs, kFaWaves * 64, 0, stream>>>(a);                 \
    if (p.splits > 1) kvq_fa_merge<DD><<<mgrid, 256, 0, stream>>>(a);           \
  } while (0)
  if (D == 256) Q35_FA(256); else if (D == 128) Q35_FA(128); else Q35_FA(64);
#undef Q35_FA
  return q35_last_error();
}
