// Append to the paged 4-bit cache with the position rotation applied on the
// way, and the read-back of what the cache holds.
//
// Rotation of a channel pair (x1, x2) at position t: (x1 c - x2 s, x2 c + x1 s)
// with c, s = cos / sin[t] in fp32; each product and each sum is rounded to
// fp32 (no FMA) and the result once to the dtype, so the stored keys do not
// depend on how a compiler contracts the expression.
//
// A call rotates q (and k where it is asked for), quantizes the tiles that
// leave the window, whose tokens are new or still in the ring, and writes the
// sink's and the window's new rows.  A row that packing reads from the ring is
// overwritten only when a call brings more than one token, so a decode step
// is a single launch, and prompts take a second one for the rows.
//
// What bounds it: rotation moves bytes (q in and out), packing is instructions
// (seven exact cuts per group, 7 packed compares and adds per pair of values),
// so their blocks alternate in one launch.  A prompt of 16384 tokens with 40 / 8
// heads in bf16, 464 MB: 95 us (4.9 TB/s; DRAM moves 420 MB of it).  Neither side
// is full there: 52% of the issue slots, 30 warps per SM of which most wait for
// loads (7.1 per instruction issued).  13 prompts of 11796 tokens, 290 MB: 58 us
// (5.0 TB/s).  A decode step: 2.6 us for one sequence, 9.0 us for 128 (5.9 MB,
// four of them completing a tile: latency of the packing blocks).  With the
// read-back: one block per token and one per (tile, head) took 140 us; eight
// tokens per rotation block 110 us, four 114, sixteen 117.
// Sharing a group's cuts over its threads took packing from 63 to 50 us,
// keeping a token's angles over its heads and exact batches of heads took
// rotation from 95 to 65 us.
#include <algorithm>

#include "innerq_internal.h"
#include "paged.cuh"

namespace innerq {
namespace {

struct NewDev {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  const int32_t* cu;  // null: one token per sequence
  const float* cos;
  const float* sin;
  int64_t cs_stride;
  uint16_t* q_out;
  uint16_t* k_out;
  int64_t qo_st, qo_sh, ko_st, ko_sh;
  int Hq, T, rot, interleaved, max_pos;
};

template <int DT> __device__ constexpr uint16_t nan16() { return DT == F16 ? 0x7e00 : 0x7fc0; }

// which sequence holds packed token t (cu[b] <= t < cu[b + 1]); all threads of
// the block take part and get the answer through *found (-1: none)
__device__ __forceinline__ void find_seq(const int32_t* cu, int B, int t, int* found) {
  if (threadIdx.x == 0) *found = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < B; b += blockDim.x)
    if (cu[b] <= t && t < cu[b + 1]) *found = b;
  __syncthreads();
}

// rotate one pair of fp32 values
__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = x;
}

// The two 8-channel chunks of unit u (0..7) of a head: rotation partners of
// each other (half-split rotation) or neighbours.
__device__ __forceinline__ void unit_chunks(const NewDev& n, int u, int& d0, int& d1) {
  const int half = n.rot >> 1;
  if (!n.interleaved && 8 * u < half) {
    d0 = 8 * u;
    d1 = d0 + half;
  } else if (!n.interleaved) {
    d0 = n.rot + 16 * (u - (n.rot >> 4));
    d1 = d0 + 8;
  } else {
    d0 = 16 * u;
    d1 = d0 + 8;
  }
}

// two fp32 values rounded to the dtype, as one word
template <int DT> __device__ __forceinline__ uint32_t round2(float lo, float hi) {
  uint32_t r;
  if constexpr (DT == F16)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// the halves of a word of the dtype as fp32
template <int DT> __device__ __forceinline__ float lo_f(uint32_t w) {
  if constexpr (DT == F16) return __low2float(as_pair<F16>(w));
  return __uint_as_float(w << 16);
}
template <int DT> __device__ __forceinline__ float hi_f(uint32_t w) {
  if constexpr (DT == F16) return __high2float(as_pair<F16>(w));
  return __uint_as_float(w & 0xffff0000u);
}

// the angles of a unit at one position
struct Angles {
  float c[8], s[8];
  enum { kNone, kHalves, kPairs, kNaN } mode;
};

__device__ __forceinline__ void load_angles(const NewDev& n, int u, int d0, int pos, Angles& g) {
  g.mode = d0 >= n.rot ? Angles::kNone
           : (unsigned)pos >= (unsigned)n.max_pos ? Angles::kNaN  // beyond the table: NaN, never a wrong angle
           : n.interleaved ? Angles::kPairs : Angles::kHalves;
  if (g.mode == Angles::kNone || g.mode == Angles::kNaN) return;
  const float4* c = reinterpret_cast<const float4*>(n.cos + pos * n.cs_stride + 8 * u);
  const float4* s = reinterpret_cast<const float4*>(n.sin + pos * n.cs_stride + 8 * u);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 c4 = __ldg(c + i), s4 = __ldg(s + i);
    g.c[4 * i] = c4.x; g.c[4 * i + 1] = c4.y; g.c[4 * i + 2] = c4.z; g.c[4 * i + 3] = c4.w;
    g.s[4 * i] = s4.x; g.s[4 * i + 1] = s4.y; g.s[4 * i + 2] = s4.z; g.s[4 * i + 3] = s4.w;
  }
}

// rotate the two chunks of a unit
template <int DT>
__device__ __forceinline__ void rotate_unit(const Angles& g, uint4& x, uint4& y) {
  uint32_t* xa = reinterpret_cast<uint32_t*>(&x);
  uint32_t* ya = reinterpret_cast<uint32_t*>(&y);
  if (g.mode == Angles::kHalves) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a0 = lo_f<DT>(xa[i]), a1 = hi_f<DT>(xa[i]), b0 = lo_f<DT>(ya[i]), b1 = hi_f<DT>(ya[i]);
      rotate(a0, b0, g.c[2 * i], g.s[2 * i]);
      rotate(a1, b1, g.c[2 * i + 1], g.s[2 * i + 1]);
      xa[i] = round2<DT>(a0, a1);
      ya[i] = round2<DT>(b0, b1);
    }
  } else if (g.mode == Angles::kPairs) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a0 = lo_f<DT>(xa[i]), a1 = hi_f<DT>(xa[i]), b0 = lo_f<DT>(ya[i]), b1 = hi_f<DT>(ya[i]);
      rotate(a0, a1, g.c[i], g.s[i]);
      rotate(b0, b1, g.c[4 + i], g.s[4 + i]);
      xa[i] = round2<DT>(a0, a1);
      ya[i] = round2<DT>(b0, b1);
    }
  } else if (g.mode == Angles::kNaN) {
#pragma unroll
    for (int i = 0; i < 4; ++i) xa[i] = ya[i] = nan16<DT>() * 0x00010001u;
  }
}

// the scale of a group from the bits of its largest magnitude
template <int DT> __device__ __forceinline__ uint16_t scale_of(uint16_t amax) {
  const float a = to_f<DT>(amax);
  return (__float_as_uint(a) & 0x7f800000u) == 0x7f800000u ? nan16<DT>() : from_f<DT>(__fdiv_rn(a, 7.f));
}

// cuts of a scale rounded up to the dtype, in both halves of a word
template <int DT> __device__ __forceinline__ void cuts_of(uint16_t scale, uint32_t* c) {
  float f[7];
  code_cuts<DT == F16 ? 10 : 7, 7>((double)to_f<DT>(scale), f);
#pragma unroll
  for (int i = 0; i < 7; ++i) c[i] = cut_bits<DT>(f[i]);
}

// the larger of two magnitudes as bits: a NaN (largest bits of all) stays
__device__ __forceinline__ uint32_t maxbits2(uint32_t a, uint32_t b) {
  return __vmaxu2(a & 0x7fff7fffu, b & 0x7fff7fffu);
}

__device__ __forceinline__ uint32_t max4(const uint4& v) {
  const uint32_t m = maxbits2(maxbits2(v.x, v.y), maxbits2(v.z, v.w));
  return max(m & 0xffff, m >> 16);
}

// The scale of a group and its seven cuts (rounded up to the dtype) as eight
// 16-bit values: cuts 0-6, then the scale.
template <int DT> __device__ __forceinline__ uint4 group_of(uint16_t amax) {
  const uint16_t scale = scale_of<DT>(amax);
  uint32_t c[7];
  cuts_of<DT>(scale, c);
  return make_uint4(c[0] | c[1] << 16, c[2] | c[3] << 16, c[4] | c[5] << 16, c[6] | (uint32_t)scale << 16);
}

constexpr int kAppendThreads = 256;  // 32 tokens x 8 units, or 64 channel pairs x 4 l

// Quantize the 32-token tile `t` (32-token units after the sink) of sequence b
// for heads h0 .. h1.  A thread is a unit (two chunks of 8 channels) of one
// token for the keys, whose angles it keeps over the heads, and 8 tokens of a
// pair of channels for the values.  Maxima meet in shared memory, one thread
// per group turns them into the group's cuts, and every thread codes its
// values against them.
template <int DT>
__device__ void pack_tile(const PagedDev& c, const NewDev& n, int b, int h0, int h1, int t, int len0, int cu0) {
  __shared__ __align__(16) uint16_t kmax[32][16];
  __shared__ uint32_t vmax[4][64];
  __shared__ uint4 kgroup[32][4], vgroup[128];
  const int first = c.w_sink + 32 * t, tid = threadIdx.x;
  const int r = tid >> 3, u = tid & 7, pos = first + r;  // keys
  const int dp = tid & 63, l = tid >> 6;                 // values
  uint8_t* blk = c.tile(b, h0, t);
  int64_t base = c.dense_base(b, h0);
  if (blk == nullptr || base < 0) return;
  int d0, d1;
  unit_chunks(n, u, d0, d1);
  const bool fresh = pos >= len0, all_fresh = first >= len0;
  Angles g;
  g.mode = Angles::kNone;
  if (fresh) load_angles(n, u, d0, pos, g);
  const int64_t tok = (int64_t)cu0 + first - len0;
  const uint16_t* row = fresh ? n.k + (tok + r) * n.k_st + h0 * n.k_sh : c.dk + base + (int64_t)c.row_of(pos) * kD;
  const int64_t row_step = fresh ? n.k_sh : (int64_t)c.dense_rows() * kD;
  const uint16_t* vrow = n.v + (tok + 2 * l) * n.v_st + h0 * n.v_sh + 2 * dp;
#pragma unroll 1
  for (int h = h0; h < h1; ++h) {
    uint4 k[2] = {*reinterpret_cast<const uint4*>(row + d0), *reinterpret_cast<const uint4*>(row + d1)};
    uint32_t vv[8], m = 0;  // nibble i: token 8 (i & 3) + 2 l + (i >> 2)
    if (all_fresh) {
      const uint16_t* p = vrow;
#pragma unroll
      for (int i = 0; i < 4; ++i, p += 8 * n.v_st) {
        vv[i] = *reinterpret_cast<const uint32_t*>(p);
        vv[i + 4] = *reinterpret_cast<const uint32_t*>(p + n.v_st);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int o = 8 * (i & 3) + 2 * l + (i >> 2);
        const uint16_t* p = first + o >= len0 ? n.v + (tok + o) * n.v_st + h * n.v_sh : c.dv + base + (int64_t)c.row_of(first + o) * kD;
        vv[i] = *reinterpret_cast<const uint32_t*>(p + 2 * dp);
      }
    }
    row += row_step;
    vrow += n.v_sh;
    base += (int64_t)c.dense_rows() * kD;
    rotate_unit<DT>(g, k[0], k[1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = maxbits2(m, vv[i]);
    kmax[r][d0 >> 3] = (uint16_t)max4(k[0]);
    kmax[r][d1 >> 3] = (uint16_t)max4(k[1]);
    vmax[l][dp] = m;
    __syncthreads();
    if (tid < 128) {
      const uint2 m4 = reinterpret_cast<const uint2*>(kmax[tid >> 2])[tid & 3];
      const uint32_t mm = maxbits2(m4.x, m4.y);
      const uint4 q = group_of<DT>((uint16_t)max(mm & 0xffff, mm >> 16));
      kgroup[tid >> 2][tid & 3] = q;
      reinterpret_cast<uint16_t*>(blk + kKScale)[((tid >> 2) & 7) * 16 + (tid >> 5) * 4 + (tid & 3)] = (uint16_t)(q.w >> 16);
    } else {
      const int d = tid - 128;
      const uint32_t mm = maxbits2(maxbits2(vmax[0][d >> 1], vmax[1][d >> 1]), maxbits2(vmax[2][d >> 1], vmax[3][d >> 1]));
      const uint4 q = group_of<DT>((uint16_t)(d & 1 ? mm >> 16 : mm & 0xffff));
      vgroup[d] = q;
      reinterpret_cast<uint16_t*>(blk + kVScale)[d] = (uint16_t)(q.w >> 16);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = i ? d1 : d0;
      const uint4 q = kgroup[r][d >> 5];
      const uint32_t cut[7] = {__byte_perm(q.x, 0, 0x1010), __byte_perm(q.x, 0, 0x3232), __byte_perm(q.y, 0, 0x1010),
                               __byte_perm(q.y, 0, 0x3232), __byte_perm(q.z, 0, 0x1010), __byte_perm(q.z, 0, 0x3232),
                               __byte_perm(q.w, 0, 0x1010)};
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&k[i]);
      uint32_t o = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t code = sym_codes2<DT, 4>(w[e], cut);
        o |= ((code & 15u) | ((code >> 12) & 0xf0u)) << (8 * e);
      }
      reinterpret_cast<uint32_t*>(blk)[(r * 4 + ((d >> 3) & 3)) * 4 + (d >> 5)] = o;
    }
    const uint4 q0 = vgroup[2 * dp], q1 = vgroup[2 * dp + 1];
    const uint32_t cut[7] = {__byte_perm(q0.x, q1.x, 0x5410), __byte_perm(q0.x, q1.x, 0x7632), __byte_perm(q0.y, q1.y, 0x5410),
                             __byte_perm(q0.y, q1.y, 0x7632), __byte_perm(q0.z, q1.z, 0x5410), __byte_perm(q0.z, q1.z, 0x7632),
                             __byte_perm(q0.w, q1.w, 0x5410)};
    uint32_t o0 = 0, o1 = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t code = sym_codes2<DT, 4>(vv[i], cut);
      o0 |= (code & 15u) << (4 * i);
      o1 |= ((code >> 16) & 15u) << (4 * i);
    }
    const int d = 2 * dp;
    reinterpret_cast<uint2*>(blk + kVCodes)[((((d >> 2) & 3) * 8 + (d >> 4)) * 4 + l) * 2 + ((d >> 1) & 1)] = make_uint2(o0, o1);
    blk += (int64_t)c.page_tiles * kBlockBytes;  // the same tile of the next head
  }
}

constexpr int kPackHeads = 2;  // heads of a pack block

template <int DT>
__device__ __forceinline__ void pack_block(const PagedDev& c, const NewDev& n, int item, int part) {
  __shared__ int sb;
  int b = item, t, len0, cu0;
  if (n.cu) {
    // items of sequence b start at cu[b] / 32 + b: room for its new tiles
    if (threadIdx.x == 0) sb = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < c.B; i += blockDim.x)
      if (n.cu[i] / 32 + i <= item && item < n.cu[i + 1] / 32 + i + 1) sb = i;
    __syncthreads();
    b = sb;
    if (b < 0) return;
    cu0 = n.cu[b];
    len0 = c.lens[b];
    t = (c.n_packed(len0) >> 5) + item - (cu0 / 32 + b);
    // a cu_seqlens that runs past the tokens given never reads past them
    if (len0 < 0 || cu0 < 0 || 32 * t >= c.n_packed(len0 + min(n.cu[b + 1], n.T) - cu0)) return;
  } else {
    cu0 = b;
    len0 = c.lens[b];
    t = c.n_packed(len0) >> 5;
    if (len0 < 0 || 32 * t >= c.n_packed(len0 + 1)) return;
  }
  pack_tile<DT>(c, n, b, part * kPackHeads, min(c.Hkv, (part + 1) * kPackHeads), t, len0, cu0);
}

// Rotate the rows of heads h0, h0 + step, .. of one token.  A thread is one
// unit of the token, keeps its angles over the heads and has the loads of
// N heads under way at a time.
template <int DT, int N>
__device__ __forceinline__ void rotate_batch(const Angles& g, int d0, int d1, const uint16_t* src, int64_t src_step, uint16_t* dst,
                                             int64_t dst_step) {
  uint4 x[N], y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = *reinterpret_cast<const uint4*>(src + i * src_step + d0);
    y[i] = *reinterpret_cast<const uint4*>(src + i * src_step + d1);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    rotate_unit<DT>(g, x[i], y[i]);
    *reinterpret_cast<uint4*>(dst + i * dst_step + d0) = x[i];
    *reinterpret_cast<uint4*>(dst + i * dst_step + d1) = y[i];
  }
}
template <int DT>
__device__ __forceinline__ void rotate_rows(const Angles& g, int d0, int d1, const uint16_t* src, int64_t src_sh, uint16_t* dst,
                                            int64_t dst_sh, int heads, int h0, int step) {
  constexpr int kBatch = 2;
  int left = heads > h0 ? (heads - h0 + step - 1) / step : 0;
  const int64_t ss = step * src_sh, ds = step * dst_sh;
  src += h0 * src_sh;
  dst += h0 * dst_sh;
#pragma unroll 1
  for (; left >= kBatch; left -= kBatch, src += kBatch * ss, dst += kBatch * ds) rotate_batch<DT, kBatch>(g, d0, d1, src, ss, dst, ds);
#pragma unroll 1
  for (; left > 0; --left, src += ss, dst += ds) rotate_batch<DT, 1>(g, d0, d1, src, ss, dst, ds);
}

// the rotated q, and k where it is asked for, of one token
template <int DT>
__device__ __forceinline__ void rotate_token(const NewDev& n, int Hkv, int tok, int pos, int h0, int step) {
  const int u = threadIdx.x & 7;
  int d0, d1;
  unit_chunks(n, u, d0, d1);
  Angles g;
  load_angles(n, u, d0, pos, g);
  rotate_rows<DT>(g, d0, d1, n.q + (int64_t)tok * n.q_st, n.q_sh, n.q_out + (int64_t)tok * n.qo_st, n.qo_sh, n.Hq, h0, step);
  if (n.k_out)
    rotate_rows<DT>(g, d0, d1, n.k + (int64_t)tok * n.k_st, n.k_sh, n.k_out + (int64_t)tok * n.ko_st, n.ko_sh, Hkv, h0, step);
}

// the rows of a token that belongs to no sequence
template <int DT>
__device__ __forceinline__ void nan_token(const NewDev& n, int Hkv, int tok, int h0, int step) {
  constexpr uint32_t nan2 = nan16<DT>() * 0x00010001u;
  const uint4 nan4 = make_uint4(nan2, nan2, nan2, nan2);
  const int d = 16 * (threadIdx.x & 7);
  auto fill = [&](uint16_t* row, int64_t sh, int heads) {
    for (int h = h0; h < heads; h += step) {
      *reinterpret_cast<uint4*>(row + h * sh + d) = nan4;
      *reinterpret_cast<uint4*>(row + h * sh + d + 8) = nan4;
    }
  };
  fill(n.q_out + (int64_t)tok * n.qo_st, n.qo_sh, n.Hq);
  if (n.k_out) fill(n.k_out + (int64_t)tok * n.ko_st, n.ko_sh, Hkv);
}

// the row that a token of the sink or the window gets in its slot
// (wait: the first head's loads come before the grid's predecessor is waited for)
template <int DT>
__device__ __forceinline__ void keep_token(const PagedDev& c, const NewDev& n, int tok, int b, int pos, int row, int h0, int step,
                                           bool wait) {
  const int u = threadIdx.x & 7;
  int d0, d1;
  unit_chunks(n, u, d0, d1);
  Angles g;
  load_angles(n, u, d0, pos, g);
  for (int h = h0; h < c.Hkv; h += step) {
    const uint16_t* p = n.k + (int64_t)tok * n.k_st + h * n.k_sh;
    const uint16_t* r = n.v + (int64_t)tok * n.v_st + h * n.v_sh;
    uint4 x = *reinterpret_cast<const uint4*>(p + d0), y = *reinterpret_cast<const uint4*>(p + d1);
    const uint4 v0 = *reinterpret_cast<const uint4*>(r + d0), v1 = *reinterpret_cast<const uint4*>(r + d1);
    rotate_unit<DT>(g, x, y);
    if (wait && h == h0) {
      griddep_wait();
      griddep_launch_dependents();
    }
    const int64_t at = c.dense_base(b, h);
    if (at < 0) return;
    uint16_t* k = c.dk + at + (int64_t)row * kD;
    uint16_t* v = c.dv + at + (int64_t)row * kD;
    *reinterpret_cast<uint4*>(k + d0) = x;
    *reinterpret_cast<uint4*>(k + d1) = y;
    *reinterpret_cast<uint4*>(v + d0) = v0;
    *reinterpret_cast<uint4*>(v + d1) = v1;
  }
}

constexpr int kTokens = 8;                                // tokens of a block of prompts, eight threads each at a time
constexpr int kTokenHeads = kAppendThreads / 8 / kTokens;  // heads that its threads take at once

// role 0: a decode step, one token per sequence; 1: prompts, rotation and
// packing; 2: prompts, the sink's and the window's rows (after the packing,
// which may read what they overwrite)
template <int DT, int ROLE>
__global__ void __launch_bounds__(kAppendThreads, 4) append_kernel(PagedDev c, NewDev n, int n_pack, int split) {
  const int blk = blockIdx.x, parts = (c.Hkv + kPackHeads - 1) / kPackHeads;
  if (ROLE == 2) {
    // Up to the wait this reads only what earlier kernels than its predecessor
    // (role 1) wrote, and they are complete: role 1 lets this grid start after
    // its own wait.
    const int groups = (c.dense_rows() + kTokens - 1) / kTokens, b = blk / groups;
    const int row = blk % groups * kTokens + ((threadIdx.x >> 3) & (kTokens - 1)), h0 = threadIdx.x / (8 * kTokens);
    const int len0 = c.lens[b], cu0 = n.cu[b], after = len0 + min(n.cu[b + 1], n.T) - cu0;
    // the position whose row this is: of the window's the one at or after its first
    const int np = c.n_packed(after), j = row - c.w_sink;
    int place = (j - np) % c.ring();
    if (place < 0) place += c.ring();
    const int pos = j < 0 ? row : c.w_sink + np + place;
    if (len0 >= 0 && cu0 >= 0 && row < c.dense_rows() && pos >= len0 && pos < after && h0 < c.Hkv) {
      keep_token<DT>(c, n, cu0 + pos - len0, b, pos, row, h0, kTokenHeads, true);
    } else {
      griddep_wait();
      griddep_launch_dependents();
    }
    return;
  }
  griddep_wait();
  griddep_launch_dependents();
  // packing (bound by instructions) and rotation (by memory) blocks alternate
  const int packs = (int)((int64_t)blk * n_pack / gridDim.x);
  if ((int)((int64_t)(blk + 1) * n_pack / gridDim.x) > packs) {
    pack_block<DT>(c, n, packs / parts, packs % parts);
    return;
  }
  const int rest = blk - packs;
  if (ROLE == 0) {  // `split` blocks share a token's heads
    const int rows = kAppendThreads / 8, tok = rest / split, len0 = c.lens[tok];
    const int h0 = (threadIdx.x >> 3) + rest % split * rows;
    if (len0 < 0) {
      nan_token<DT>(n, c.Hkv, tok, h0, rows * split);
      return;
    }
    rotate_token<DT>(n, c.Hkv, tok, len0, h0, rows * split);
    keep_token<DT>(c, n, tok, tok, len0, c.row_of(len0), h0, rows * split, false);
    return;
  }
  __shared__ int sb;
  const int tok0 = rest * kTokens, tok = tok0 + ((threadIdx.x >> 3) & (kTokens - 1));
  find_seq(n.cu, c.B, tok0, &sb);
  int b = max(sb, 0);
  while (b < c.B && tok >= n.cu[b + 1]) ++b;
  if (tok >= n.T) return;
  const int len0 = b < c.B ? c.lens[b] : -1, cu0 = b < c.B ? n.cu[b] : 0, h0 = threadIdx.x / (8 * kTokens);
  if (len0 < 0 || tok < cu0)
    nan_token<DT>(n, c.Hkv, tok, h0, kTokenHeads);
  else
    rotate_token<DT>(n, c.Hkv, tok, len0 + tok - cu0, h0, kTokenHeads);
}

// (u - 8) s of the codes in bits 0-3 and 16-19 of w: exact in the dtype before
// the one rounding of the product, as the fp32 product of the definition
template <int DT> __device__ __forceinline__ uint32_t value2(uint32_t w, uint32_t s2) {
  constexpr uint32_t magic = DT == F16 ? 0x64006400u : 0x43004300u;  // 1024, 128: the code is the last digits
  constexpr uint32_t bias = DT == F16 ? 0x64086408u : 0x43084308u;
  const auto c = __hsub2(as_pair<DT>((w & 0x000f000fu) | magic), as_pair<DT>(bias));
  return pair_bits<DT>(__hmul2(c, as_pair<DT>(s2)));
}

// Read-back: one block per head and tile of 32 positions.  Sink, packed part and
// window begin and end at multiples of 32, so a tile is of one kind.
// The windows of 128 sequences (16 bits, 8 heads, 127 MB): 24 us (5.3 TB/s);
// 16384 packed tokens of one (86 MB): 17.7 us (4.9 TB/s).  Loads bound it (9.6 and
// 5.8 warps wait for them per instruction issued) and, for packed tokens, 56% of
// the issue slots.
template <int DT>
__global__ void __launch_bounds__(128, 8)
    read_kernel(PagedDev c, const int32_t* starts, const int32_t* cu, int n_tokens, uint16_t* ko, uint16_t* vo) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int sb;
  const int item = blockIdx.x / c.Hkv, h = blockIdx.x % c.Hkv, tid = threadIdx.x;
  // items of sequence b start at cu[b] / 32 + 2 b: room for tiles cut at both ends
  if (tid == 0) sb = -1;
  __syncthreads();
  for (int i = tid; i < c.B; i += 128)
    if (cu[i] / 32 + 2 * i <= item && item < cu[i + 1] / 32 + 2 * i + 2) sb = i;
  __syncthreads();
  const int b = sb;
  if (b < 0) return;
  const int cu0 = cu[b], count = min(cu[b + 1], n_tokens) - cu0, start = starts[b], len = c.lens[b];
  if (cu0 < 0 || count <= 0) return;
  const int p0 = (start >= 0 ? start & ~31 : -((-start + 31) & ~31)) + 32 * (item - (cu0 / 32 + 2 * b));
  if (p0 >= start + count) return;
  // position p of the tile goes to row cu0 - start + p, if start <= p < start + count
  const int64_t pitch = (int64_t)c.Hkv * kD, out0 = ((int64_t)cu0 - start + p0) * pitch;
  const int lo = start - p0, hi = start + count - p0;
  auto put = [&](uint16_t* o, int r, int d, uint4 v) {
    if (r >= lo && r < hi) *reinterpret_cast<uint4*>(o + r * pitch + d) = v;
  };
  constexpr uint32_t nan2 = nan16<DT>() * 0x00010001u;
  const uint4 nan4 = make_uint4(nan2, nan2, nan2, nan2);
  const int u0 = p0 - c.w_sink;
  const bool packed = u0 >= 0 && u0 < c.n_packed(len);
  const int row = packed || p0 < 0 ? 0 : c.row_of(p0);
  uint16_t* kr = ko + out0 + h * kD;
  uint16_t* vr = vo + out0 + h * kD;
  const uint8_t* blk = packed ? c.tile(b, h, u0 >> 5) : nullptr;
  const int64_t base = packed ? -1 : c.dense_base(b, h);
  if (p0 < 0 || p0 >= len || (packed ? blk == nullptr : base < 0)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      put(kr, 8 * i + (tid >> 4), 8 * (tid & 15), nan4);
      put(vr, 8 * i + (tid >> 4), 8 * (tid & 15), nan4);
    }
  } else if (!packed) {
    const int64_t at = base + (int64_t)row * kD;
    uint4 k[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (tid >> 4), d = 8 * (tid & 15);
      const bool in = p0 + r < len && r >= lo && r < hi;
      k[i] = in ? *reinterpret_cast<const uint4*>(c.dk + at + r * kD + d) : nan4;
      v[i] = in ? *reinterpret_cast<const uint4*>(c.dv + at + r * kD + d) : nan4;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      put(kr, 8 * i + (tid >> 4), 8 * (tid & 15), k[i]);
      put(vr, 8 * i + (tid >> 4), 8 * (tid & 15), v[i]);
    }
  } else {
    // keys: token r, channels 32 g + 8 l ..; values: channels 4 q .., tokens 8 (n & 3) + 2 vl + (n >> 2)
    const int r = tid >> 2, l = tid & 3, vl = tid >> 5, q = tid & 31;
    const uint4 kw = reinterpret_cast<const uint4*>(blk)[tid];
    const uint4 vw = reinterpret_cast<const uint4*>(blk + kVCodes)[((q & 3) * 8 + (q >> 2)) * 4 + vl];
    const uint2 ks = reinterpret_cast<const uint2*>(blk + kKScale)[(r & 7) * 4 + (r >> 3)];
    const uint2 vs = reinterpret_cast<const uint2*>(blk + kVScale)[q];
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&kw);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint32_t s2 = __byte_perm(g & 2 ? ks.y : ks.x, 0, g & 1 ? 0x3232 : 0x1010);
      uint32_t e[4];  // channels (x, x + 4)
#pragma unroll
      for (int x = 0; x < 4; ++x) e[x] = value2<DT>(w[g] >> (4 * x), s2);
      put(kr, r, 32 * g + 8 * l,
          make_uint4(__byte_perm(e[0], e[1], 0x5410), __byte_perm(e[2], e[3], 0x5410), __byte_perm(e[0], e[1], 0x7632),
                     __byte_perm(e[2], e[3], 0x7632)));
    }
    w = reinterpret_cast<const uint32_t*>(&vw);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      uint32_t e[4];  // channel y of tokens 8 x + 2 vl and the one after it
#pragma unroll
      for (int y = 0; y < 4; ++y)
        e[y] = value2<DT>(w[y] >> (4 * x), __byte_perm(y & 2 ? vs.y : vs.x, 0, y & 1 ? 0x3232 : 0x1010));
      const int t = 8 * x + 2 * vl;
      if (t >= lo && t < hi)
        *reinterpret_cast<uint2*>(vr + t * pitch + 4 * q) =
            make_uint2(__byte_perm(e[0], e[1], 0x5410), __byte_perm(e[2], e[3], 0x5410));
      if (t + 1 >= lo && t + 1 < hi)
        *reinterpret_cast<uint2*>(vr + (t + 1) * pitch + 4 * q) =
            make_uint2(__byte_perm(e[0], e[1], 0x7632), __byte_perm(e[2], e[3], 0x7632));
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int cuda_rc(cudaError_t e, const char* what) {
  return e == cudaSuccess ? INNERQ_OK : set_last_error(INNERQ_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// pack blocks of a call: an upper bound of the tiles it can complete, by heads
int64_t pack_blocks(const PagedDev& c, const NewDev& n) {
  const int64_t items = n.cu ? n.T / 32 + c.B : c.B;
  return items * ((c.Hkv + kPackHeads - 1) / kPackHeads);
}

template <int DT>
cudaError_t launch_append(const PagedDev& c, const NewDev& n, cudaStream_t s) {
  const int n_pack = (int)pack_blocks(c, n);
  const dim3 block(kAppendThreads);
  if (n.cu == nullptr) {
    // few tokens: several blocks per token, so that a thread has one row
    const int per = kAppendThreads / 8, split = n.T < 256 ? (std::max(n.Hq, c.Hkv) + per - 1) / per : 1;
    return launch_pdl(append_kernel<DT, 0>, dim3(n_pack + n.T * split), block, 0, s, c, n, n_pack, split);
  }
  const int n_rotate = (n.T + kTokens - 1) / kTokens, rows = c.w_sink + c.w_recent + 32;
  cudaError_t e = launch_pdl(append_kernel<DT, 1>, dim3(n_pack + n_rotate), block, 0, s, c, n, n_pack, 1);
  if (e != cudaSuccess || c.B == 0) return e;
  return launch_pdl(append_kernel<DT, 2>, dim3(c.B * ((rows + kTokens - 1) / kTokens)), block, 0, s, c, n, 0, 1);
}

}  // namespace

int paged_dev(const innerq_paged* c, PagedDev& d) {
  if (!c) return set_last_error(INNERQ_ERR_ARG, "null cache");
  if (c->struct_size != (int32_t)sizeof(innerq_paged))
    return set_last_error(INNERQ_ERR_ARG, "struct_size %d != %d (ABI mismatch)", c->struct_size, (int)sizeof(innerq_paged));
  if (c->dtype != INNERQ_DT_F16 && c->dtype != INNERQ_DT_BF16) return set_last_error(INNERQ_ERR_ARG, "dtype %d", c->dtype);
  if (c->D != kD) return set_last_error(INNERQ_ERR_UNSUPPORTED, "head_dim %d (only 128 is built)", c->D);
  if (c->Hkv <= 0 || c->n_pages < 0 || c->n_slots < 0 || c->B < 0 || c->max_pages < 0)
    return set_last_error(INNERQ_ERR_ARG, "negative size");
  if (c->page_tiles < 1 || c->page_tiles > 64)
    return set_last_error(INNERQ_ERR_ARG, "a page holds %d tiles (1 to 64)", c->page_tiles);
  if (c->w_sink < 0 || c->w_recent < 0 || c->w_sink % 32 || c->w_recent % 32 || c->w_sink > 4096 || c->w_recent > 4096)
    return set_last_error(INNERQ_ERR_ARG, "sink %d and recent window %d must be multiples of 32 up to 4096", c->w_sink, c->w_recent);
  if (c->B > 0 && (!c->slots || !c->seq_lens || !c->dense_k || !c->dense_v))
    return set_last_error(INNERQ_ERR_ARG, "null pointer");
  // the table is read before a page number is compared with n_pages
  if (c->B > 0 && c->max_pages > 0 && (!c->table || (c->n_pages > 0 && !c->pages)))
    return set_last_error(INNERQ_ERR_ARG, "null pages or page table");
  if (!aligned16(c->pages) || !aligned16(c->dense_k) || !aligned16(c->dense_v))
    return set_last_error(INNERQ_ERR_ARG, "pages and slots must be 16-byte aligned");
  d.pages = (uint8_t*)c->pages;
  d.dk = (uint16_t*)c->dense_k;
  d.dv = (uint16_t*)c->dense_v;
  d.table = c->table;
  d.slots = c->slots;
  d.lens = c->seq_lens;
  d.table_stride = c->table_stride;
  d.B = c->B; d.Hkv = c->Hkv; d.page_tiles = c->page_tiles;
  d.n_pages = c->n_pages; d.n_slots = c->n_slots;
  d.w_sink = c->w_sink; d.w_recent = c->w_recent; d.max_pages = c->max_pages;
  return INNERQ_OK;
}

}  // namespace innerq

using namespace innerq;

extern "C" int innerq_paged_append(const innerq_paged* cache, const innerq_paged_new* a, void* stream) {
  PagedDev c;
  if (int rc = paged_dev(cache, c)) return rc;
  if (!a || a->struct_size != (int32_t)sizeof(innerq_paged_new))
    return set_last_error(INNERQ_ERR_ARG, "struct_size of the new tokens (ABI mismatch)");
  if (a->Hq < 0 || a->T < 0) return set_last_error(INNERQ_ERR_ARG, "negative size");
  if (!a->cu_seqlens && a->T != c.B)
    return set_last_error(INNERQ_ERR_ARG, "%d tokens for %d sequences need cu_seqlens", a->T, c.B);
  if (a->rot_dim < 0 || a->rot_dim > kD || a->rot_dim % 16)
    return set_last_error(INNERQ_ERR_ARG, "rotation over %d channels (a multiple of 16 up to 128)", a->rot_dim);
  if (a->T == 0) return INNERQ_OK;
  if (!a->k || !a->v || (a->Hq > 0 && (!a->q || !a->q_out))) return set_last_error(INNERQ_ERR_ARG, "null pointer");
  if (a->rot_dim && (!a->cos || !a->sin || a->max_pos <= 0)) return set_last_error(INNERQ_ERR_ARG, "no rotation table");
  const int64_t st[] = {a->q_st, a->q_sh, a->k_st, a->k_sh, a->v_st, a->v_sh, a->qo_st, a->qo_sh, a->ko_st, a->ko_sh};
  for (int64_t x : st)
    if (x % 8) return set_last_error(INNERQ_ERR_ARG, "strides must be multiples of 8 elements");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q_out) || !aligned16(a->k_out) ||
      (a->rot_dim && (!aligned16(a->cos) || !aligned16(a->sin) || a->cs_stride % 4)))
    return set_last_error(INNERQ_ERR_ARG, "rows must be 16-byte aligned");
  NewDev n;
  n.q = (const uint16_t*)a->q; n.k = (const uint16_t*)a->k; n.v = (const uint16_t*)a->v;
  n.q_st = a->q_st; n.q_sh = a->q_sh; n.k_st = a->k_st; n.k_sh = a->k_sh; n.v_st = a->v_st; n.v_sh = a->v_sh;
  n.cu = a->cu_seqlens;
  n.cos = a->cos; n.sin = a->sin; n.cs_stride = a->cs_stride;
  n.q_out = (uint16_t*)a->q_out; n.k_out = (uint16_t*)a->k_out;
  n.qo_st = a->qo_st; n.qo_sh = a->qo_sh; n.ko_st = a->ko_st; n.ko_sh = a->ko_sh;
  n.Hq = a->Hq; n.T = a->T; n.rot = a->rot_dim; n.interleaved = a->interleaved; n.max_pos = a->max_pos;
  if (pack_blocks(c, n) + (int64_t)a->T * 64 > 0x7fffffff || (int64_t)c.B * 4096 > 0x7fffffff)
    return set_last_error(INNERQ_ERR_ARG, "too many tokens for one launch");
  const cudaStream_t s = (cudaStream_t)stream;
  return cuda_rc(cache->dtype == INNERQ_DT_BF16 ? launch_append<BF16>(c, n, s) : launch_append<F16>(c, n, s), "paged_append");
}

extern "C" int innerq_paged_read(const innerq_paged* cache, const int32_t* starts, const int32_t* cu_seqlens, int n_tokens,
                                 void* k_out, void* v_out, void* stream) {
  PagedDev c;
  if (int rc = paged_dev(cache, c)) return rc;
  if (n_tokens < 0) return set_last_error(INNERQ_ERR_ARG, "negative size");
  if (c.B == 0 || n_tokens == 0) return INNERQ_OK;
  if (!starts || !cu_seqlens || !k_out || !v_out || !aligned16(k_out) || !aligned16(v_out))
    return set_last_error(INNERQ_ERR_ARG, "null or unaligned pointer");
  const cudaStream_t s = (cudaStream_t)stream;
  uint16_t* ko = (uint16_t*)k_out;
  uint16_t* vo = (uint16_t*)v_out;
  const int64_t blocks = ((int64_t)n_tokens / 32 + 2ll * c.B) * c.Hkv;
  if (blocks > 0x7fffffff) return set_last_error(INNERQ_ERR_ARG, "too many tokens for one launch");
  const dim3 grid((unsigned)blocks), block(128);
  return cuda_rc(cache->dtype == INNERQ_DT_BF16
                     ? launch_pdl(read_kernel<BF16>, grid, block, 0, s, c, starts, cu_seqlens, n_tokens, ko, vo)
                     : launch_pdl(read_kernel<F16>, grid, block, 0, s, c, starts, cu_seqlens, n_tokens, ko, vo),
                 "paged_read");
}
