// Append to the paged 4-bit cache with the position rotation applied on the
// way, and the read-back of what the cache holds.
//
// Rotation of a channel pair (x1, x2) at position t: (x1 c - x2 s, x2 c + x1 s)
// with c, s = cos / sin[t] in fp32; each product and each sum is rounded to
// fp32 (no FMA) and the result once to the dtype, so the stored keys do not
// depend on how a compiler contracts the expression.
//
// A call does two things: "dense" rotates q (and k) and writes the sink's and
// the window's tokens; "pack" quantizes the tiles that leave the window, whose
// tokens are new or still in the ring.  Ring rows that pack reads are
// overwritten by dense only when a call brings more than one token, so one
// token per sequence takes a single launch with both kinds of blocks and
// prompts take two launches, pack first.
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

template <int DT>
__device__ __forceinline__ void rotate_unit(const NewDev& n, int u, int d0, int pos, uint4& x, uint4& y) {
  if (n.rot == 0) return;
  if (d0 >= n.rot) return;
  uint32_t* xa = reinterpret_cast<uint32_t*>(&x);
  uint32_t* ya = reinterpret_cast<uint32_t*>(&y);
  if ((unsigned)pos >= (unsigned)n.max_pos) {  // beyond the table: NaN, never a wrong angle
    const uint32_t nan2 = nan16<DT>() * 0x00010001u;
#pragma unroll
    for (int i = 0; i < 4; ++i) xa[i] = ya[i] = nan2;
    return;
  }
  const float* c = n.cos + pos * n.cs_stride + 8 * u;
  const float* s = n.sin + pos * n.cs_stride + 8 * u;
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 c4 = __ldg(reinterpret_cast<const float4*>(c) + i);
    const float4 s4 = __ldg(reinterpret_cast<const float4*>(s) + i);
    cs[4 * i] = c4.x; cs[4 * i + 1] = c4.y; cs[4 * i + 2] = c4.z; cs[4 * i + 3] = c4.w;
    sn[4 * i] = s4.x; sn[4 * i + 1] = s4.y; sn[4 * i + 2] = s4.z; sn[4 * i + 3] = s4.w;
  }
  if (!n.interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a0 = to_f<DT>(xa[i] & 0xffff), a1 = to_f<DT>(xa[i] >> 16);
      float b0 = to_f<DT>(ya[i] & 0xffff), b1 = to_f<DT>(ya[i] >> 16);
      rotate(a0, b0, cs[2 * i], sn[2 * i]);
      rotate(a1, b1, cs[2 * i + 1], sn[2 * i + 1]);
      xa[i] = pack2(from_f<DT>(a0), from_f<DT>(a1));
      ya[i] = pack2(from_f<DT>(b0), from_f<DT>(b1));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a = to_f<DT>(xa[i] & 0xffff), b = to_f<DT>(xa[i] >> 16);
      rotate(a, b, cs[i], sn[i]);
      xa[i] = pack2(from_f<DT>(a), from_f<DT>(b));
      a = to_f<DT>(ya[i] & 0xffff), b = to_f<DT>(ya[i] >> 16);
      rotate(a, b, cs[4 + i], sn[4 + i]);
      ya[i] = pack2(from_f<DT>(a), from_f<DT>(b));
    }
  }
}

// One 8-channel chunk d0.. of a rotated key (the partner chunk is read too).
template <int DT>
__device__ __forceinline__ uint4 key_chunk(const NewDev& n, const uint16_t* row, int d0, int pos) {
  const int half = n.rot >> 1;
  if (d0 >= n.rot) return *reinterpret_cast<const uint4*>(row + d0);
  if (n.interleaved) {
    const int u = d0 >> 4;
    uint4 x = *reinterpret_cast<const uint4*>(row + 16 * u), y = *reinterpret_cast<const uint4*>(row + 16 * u + 8);
    rotate_unit<DT>(n, u, 16 * u, pos, x, y);
    return (d0 & 8) ? y : x;
  }
  const int u = (d0 < half ? d0 : d0 - half) >> 3;
  uint4 x = *reinterpret_cast<const uint4*>(row + 8 * u), y = *reinterpret_cast<const uint4*>(row + 8 * u + half);
  rotate_unit<DT>(n, u, 8 * u, pos, x, y);
  return d0 < half ? x : y;
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

// quantize the 32-token tile `t` (32-token units after the sink) of sequence
// b, head h; 128 threads
template <int DT>
__device__ void pack_tile(const PagedDev& c, const NewDev& n, int b, int h, int t, int len0, int cu0) {
  uint8_t* blk = c.tile(b, h, t);
  const int64_t base = c.dense_base(b, h);
  if (blk == nullptr || base < 0) return;
  const int first = c.w_sink + 32 * t;
  const int tid = threadIdx.x;
  __shared__ uint32_t vmax[2][64];
  {  // keys: one thread per (token, group of 32 channels)
    const int r = tid >> 2, g = tid & 3, pos = first + r;
    uint4 x[4];
    if (pos >= len0) {
      const uint16_t* row = n.k + (int64_t)(cu0 + pos - len0) * n.k_st + h * n.k_sh;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = key_chunk<DT>(n, row, 32 * g + 8 * i, pos);
    } else {
      const uint4* row = reinterpret_cast<const uint4*>(c.dk + base + (int64_t)c.row_of(pos) * kD + 32 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = row[i];
    }
    const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = maxbits2(m, w[i]);
    const uint16_t scale = scale_of<DT>(max(m & 0xffff, m >> 16));
    uint32_t cut[7];
    cuts_of<DT>(scale, cut);
#pragma unroll
    for (int i = 0; i < 7; ++i) cut[i] *= 0x00010001u;
    uint32_t* words = reinterpret_cast<uint32_t*>(blk);
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      uint32_t o = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = sym_codes2<DT, 4>(w[4 * l + i], cut);
        o |= ((u & 15u) | ((u >> 12) & 0xf0u)) << (8 * i);
      }
      words[(r * 4 + l) * 4 + g] = o;
    }
    reinterpret_cast<uint16_t*>(blk + kKScale)[(r & 7) * 16 + (r >> 3) * 4 + g] = scale;
  }
  {  // values: two threads per pair of channels, each with the 16 tokens of two l
    const int dp = tid & 63, th = tid >> 6;
    uint32_t x[16];  // [n & 3][token within the four]
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int pos = first + 8 * a + 4 * th + e;
        const uint16_t* row = pos >= len0 ? n.v + (int64_t)(cu0 + pos - len0) * n.v_st + h * n.v_sh
                                          : c.dv + base + (int64_t)c.row_of(pos) * kD;
        x[4 * a + e] = *reinterpret_cast<const uint32_t*>(row + 2 * dp);
      }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = maxbits2(m, x[i]);
    vmax[th][dp] = m;
    __syncthreads();
    m = maxbits2(m, vmax[th ^ 1][dp]);
    const uint16_t s0 = scale_of<DT>(m & 0xffff), s1 = scale_of<DT>(m >> 16);
    uint32_t cut[7], cut1[7];
    cuts_of<DT>(s0, cut);
    cuts_of<DT>(s1, cut1);
#pragma unroll
    for (int i = 0; i < 7; ++i) cut[i] |= cut1[i] << 16;
    const int d = 2 * dp, i8 = d >> 4, p = (d >> 2) & 3, mm = (d >> 1) & 1;
#pragma unroll
    for (int ll = 0; ll < 2; ++ll) {
      uint32_t o0 = 0, o1 = 0;
#pragma unroll
      for (int nn = 0; nn < 8; ++nn) {
        const uint32_t u = sym_codes2<DT, 4>(x[4 * (nn & 3) + 2 * ll + (nn >> 2)], cut);
        o0 |= (u & 15u) << (4 * nn);
        o1 |= ((u >> 16) & 15u) << (4 * nn);
      }
      uint2* words = reinterpret_cast<uint2*>(blk + kVCodes);
      words[((p * 8 + i8) * 4 + 2 * th + ll) * 2 + mm] = make_uint2(o0, o1);
    }
    if (th == 0) reinterpret_cast<uint32_t*>(blk + kVScale)[dp] = pack2(s0, s1);
  }
}

template <int DT>
__device__ __forceinline__ void pack_block(const PagedDev& c, const NewDev& n, int item, int h) {
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
  pack_tile<DT>(c, n, b, h, t, len0, cu0);
}

// rotate and store the q, k and v rows of one token
template <int DT>
__device__ __forceinline__ void dense_token(const PagedDev& c, const NewDev& n, int tok, int b, int pos, int after) {
  const bool keep = pos < c.w_sink || pos >= c.w_sink + c.n_packed(after);
  const int heads = n.Hq + 2 * c.Hkv;
  for (int i = threadIdx.x; i < heads * 8; i += blockDim.x) {
    const int row = i >> 3, u = i & 7;
    int d0, d1;
    unit_chunks(n, u, d0, d1);
    if (row < n.Hq) {
      const uint16_t* src = n.q + (int64_t)tok * n.q_st + row * n.q_sh;
      uint4 x = *reinterpret_cast<const uint4*>(src + d0), y = *reinterpret_cast<const uint4*>(src + d1);
      rotate_unit<DT>(n, u, d0, pos, x, y);
      uint16_t* dst = n.q_out + (int64_t)tok * n.qo_st + row * n.qo_sh;
      *reinterpret_cast<uint4*>(dst + d0) = x;
      *reinterpret_cast<uint4*>(dst + d1) = y;
      continue;
    }
    const bool is_k = row < n.Hq + c.Hkv;
    const int h = row - n.Hq - (is_k ? 0 : c.Hkv);
    if (!keep && !(is_k && n.k_out)) continue;
    const uint16_t* src = is_k ? n.k + (int64_t)tok * n.k_st + h * n.k_sh : n.v + (int64_t)tok * n.v_st + h * n.v_sh;
    uint4 x = *reinterpret_cast<const uint4*>(src + d0), y = *reinterpret_cast<const uint4*>(src + d1);
    if (is_k) rotate_unit<DT>(n, u, d0, pos, x, y);
    if (is_k && n.k_out) {
      uint16_t* dst = n.k_out + (int64_t)tok * n.ko_st + h * n.ko_sh;
      *reinterpret_cast<uint4*>(dst + d0) = x;
      *reinterpret_cast<uint4*>(dst + d1) = y;
    }
    const int64_t base = c.dense_base(b, h);
    if (keep && base >= 0) {
      uint16_t* dst = (is_k ? c.dk : c.dv) + base + (int64_t)c.row_of(pos) * kD;
      *reinterpret_cast<uint4*>(dst + d0) = x;
      *reinterpret_cast<uint4*>(dst + d1) = y;
    }
  }
}

// role 0: both (one token per sequence); 1: pack; 2: dense
template <int DT, int ROLE>
__global__ void __launch_bounds__(128) append_kernel(PagedDev c, NewDev n, int n_pack) {
  griddep_wait();
  griddep_launch_dependents();
  const int blk = blockIdx.x;
  if (ROLE == 1 || (ROLE == 0 && blk < n_pack)) {
    pack_block<DT>(c, n, blk / c.Hkv, blk % c.Hkv);
    return;
  }
  const int tok = ROLE == 0 ? blk - n_pack : blk;
  if (ROLE == 0) {
    const int len0 = c.lens[tok];
    if (len0 >= 0) dense_token<DT>(c, n, tok, tok, len0, len0 + 1);
    return;
  }
  __shared__ int sb;
  find_seq(n.cu, c.B, tok, &sb);
  const int b = sb;
  if (b < 0 || c.lens[b] < 0) return;
  const int len0 = c.lens[b], cu0 = n.cu[b];
  dense_token<DT>(c, n, tok, b, len0 + tok - cu0, len0 + min(n.cu[b + 1], n.T) - cu0);
}

// read-back: one block per token
template <int DT>
__global__ void __launch_bounds__(128) read_kernel(PagedDev c, const int32_t* starts, const int32_t* cu, uint16_t* ko,
                                                   uint16_t* vo) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int sb;
  const int tok = blockIdx.x;
  find_seq(cu, c.B, tok, &sb);
  const int b = sb;
  if (b < 0) return;
  const int len = c.lens[b], pos = starts[b] + tok - cu[b], u = pos - c.w_sink;
  const bool inside = pos >= 0 && pos < len, packed = u >= 0 && u < c.n_packed(len);
  for (int i = threadIdx.x; i < c.Hkv * 32; i += blockDim.x) {
    const int h = i >> 5, side = (i >> 4) & 1, d0 = 8 * (i & 15);
    uint4 o;
    uint16_t* e = reinterpret_cast<uint16_t*>(&o);
#pragma unroll
    for (int x = 0; x < 8; ++x) e[x] = nan16<DT>();
    if (inside && !packed) {
      const int64_t base = c.dense_base(b, h);
      if (base >= 0)
        o = *reinterpret_cast<const uint4*>((side ? c.dv : c.dk) + base + (int64_t)c.row_of(pos) * kD + d0);
    } else if (inside) {
      const uint8_t* blk = c.tile(b, h, u >> 5);
      const int r = u & 31;
      if (blk != nullptr && side == 0) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(blk)[(r * 4 + ((d0 >> 3) & 3)) * 4 + (d0 >> 5)];
        const float s = to_f<DT>(reinterpret_cast<const uint16_t*>(blk + kKScale)[(r & 7) * 16 + (r >> 3) * 4 + (d0 >> 5)]);
#pragma unroll
        for (int x = 0; x < 8; ++x) e[x] = from_f<DT>((float)((int)((w >> (4 * x)) & 15u) - 8) * s);
      } else if (blk != nullptr) {
        const int nib = (r >> 3) + 4 * (r & 1), l = (r >> 1) & 3, i8 = d0 >> 4, p = (d0 >> 2) & 3;
        const uint4 s4 = *reinterpret_cast<const uint4*>(blk + kVScale + 2 * d0);
        const uint16_t* s = reinterpret_cast<const uint16_t*>(&s4);
#pragma unroll
        for (int hp = 0; hp < 2; ++hp) {
          const uint4 w4 = reinterpret_cast<const uint4*>(blk + kVCodes)[((p + hp) * 8 + i8) * 4 + l];
          const uint32_t* w = reinterpret_cast<const uint32_t*>(&w4);
#pragma unroll
          for (int x = 0; x < 4; ++x)
            e[4 * hp + x] = from_f<DT>((float)((int)((w[x] >> (4 * nib)) & 15u) - 8) * to_f<DT>(s[4 * hp + x]));
        }
      }
    }
    *reinterpret_cast<uint4*>((side ? vo : ko) + ((int64_t)tok * c.Hkv + h) * kD + d0) = o;
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int cuda_rc(cudaError_t e, const char* what) {
  return e == cudaSuccess ? INNERQ_OK : set_last_error(INNERQ_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

template <int DT>
cudaError_t launch_append(const PagedDev& c, const NewDev& n, cudaStream_t s) {
  if (n.cu == nullptr) {
    const int n_pack = c.B * c.Hkv;
    return launch_pdl(append_kernel<DT, 0>, dim3(n_pack + n.T), dim3(128), 0, s, c, n, n_pack);
  }
  const int64_t items = (int64_t)(n.T / 32 + c.B) * c.Hkv;
  cudaError_t e = launch_pdl(append_kernel<DT, 1>, dim3((unsigned)items), dim3(128), 0, s, c, n, (int)items);
  if (e != cudaSuccess) return e;
  return launch_pdl(append_kernel<DT, 2>, dim3(n.T), dim3(128), 0, s, c, n, 0);
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
  if (c->n_pages > 0 && c->max_pages > 0 && (!c->pages || !c->table)) return set_last_error(INNERQ_ERR_ARG, "null pages or page table");
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
  if (c.B == 0 || a->T == 0) return INNERQ_OK;
  if (!a->k || !a->v || (a->Hq > 0 && (!a->q || !a->q_out))) return set_last_error(INNERQ_ERR_ARG, "null pointer");
  if (a->rot_dim && (!a->cos || !a->sin || a->max_pos <= 0)) return set_last_error(INNERQ_ERR_ARG, "no rotation table");
  const int64_t st[] = {a->q_st, a->q_sh, a->k_st, a->k_sh, a->v_st, a->v_sh, a->qo_st, a->qo_sh, a->ko_st, a->ko_sh};
  for (int64_t x : st)
    if (x % 8) return set_last_error(INNERQ_ERR_ARG, "strides must be multiples of 8 elements");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q_out) || !aligned16(a->k_out) ||
      (a->rot_dim && (!aligned16(a->cos) || !aligned16(a->sin) || a->cs_stride % 4)))
    return set_last_error(INNERQ_ERR_ARG, "rows must be 16-byte aligned");
  const int64_t items = (int64_t)(a->T / 32 + c.B) * c.Hkv;
  if (items + a->T > 0x7fffffff) return set_last_error(INNERQ_ERR_ARG, "too many tokens for one launch");
  NewDev n;
  n.q = (const uint16_t*)a->q; n.k = (const uint16_t*)a->k; n.v = (const uint16_t*)a->v;
  n.q_st = a->q_st; n.q_sh = a->q_sh; n.k_st = a->k_st; n.k_sh = a->k_sh; n.v_st = a->v_st; n.v_sh = a->v_sh;
  n.cu = a->cu_seqlens;
  n.cos = a->cos; n.sin = a->sin; n.cs_stride = a->cs_stride;
  n.q_out = (uint16_t*)a->q_out; n.k_out = (uint16_t*)a->k_out;
  n.qo_st = a->qo_st; n.qo_sh = a->qo_sh; n.ko_st = a->ko_st; n.ko_sh = a->ko_sh;
  n.Hq = a->Hq; n.T = a->T; n.rot = a->rot_dim; n.interleaved = a->interleaved; n.max_pos = a->max_pos;
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
  return cuda_rc(cache->dtype == INNERQ_DT_BF16
                     ? launch_pdl(read_kernel<BF16>, dim3(n_tokens), dim3(128), 0, s, c, starts, cu_seqlens, ko, vo)
                     : launch_pdl(read_kernel<F16>, dim3(n_tokens), dim3(128), 0, s, c, starts, cu_seqlens, ko, vo),
                 "paged_read");
}
