// Decode attention over the paged 4-bit cache: one query token per sequence, a
// length per sequence, one pass over 32-token tiles that may be split anywhere.
//
// Mathematics.  A 4-bit code u (0..15, offset 8) placed in the mantissa of a
// 16-bit word IS the fp16 subnormal u 2^-24 (u 2^-20 four bits higher), so one
// AND expands two codes into an fp16 tensor-core operand, exactly:
//   q.k_t = sum_g s_tg (sum_{d in g} q_d u_td - 8 sum_{d in g} q_d)
//   out_d = sum_tiles s_gd (sum_t p_t u_td - 8 sum_t p_t) / sum_t p_t
// The inner sums are mma.m16n8k16 (codes as A: 16 tokens, or 16 channels, by
// 8 query heads) with fp32 accumulators that start at the offset term; group
// scales are applied in fp32.  The query is scaled per head by a power of two
// into [2^14, 2^15) (channels below 2^-24 of the largest lose bits as fp16);
// the slots whose codes sit four bits higher take q / 16.  A probability is
// 2^8 p, relative to a running maximum that may lag by 2^7, rounded to fp16
// (11 bits down to 2^-22), as an fp16 operand takes it; with fp16 inputs that
// adds as much error again as rounding the output does (a second part for what
// it leaves took an earlier state of the kernel from 216 us to 249 on the case
// below).  The sum that divides the result is taken over the rounded values.
//   An MMA aligns its products by the operands' nominal exponents, 2^-14 for a
// subnormal, and cuts what lies some 26 bits below the largest off, towards
// zero.  Over tens of thousands of tokens that adds up along the values' scales
// unless it stays far below the probabilities' own last bits.  The values' codes
// therefore sit four bits up throughout: the cut is at 2^-20 of the tile's
// largest probability then, and the offset 8 sum p, an MMA against the code 8,
// loses what a zero value does.  At 33000 and 131000 tokens the part of the error
// that has a sign is at most 2e-5 of the output (the output's own rounding to
// fp16: 2e-4) for values normal, uniform, of one sign, constant and with one
// outlier per group; ordinary numbers u - 8 as operands do no better and take
// 256 us where this takes 227.  With the low codes where they lie (217 us) the
// cut is at 2^-16, the outliers' error was up to 4.5 times the rounding, and no
// constant in place of the 8 helps all of them.  Logits keep the cheaper form:
// only products with channels below a 64th of the query's largest are cut, and
// what is lost has the query's signs.  Log-sum-exps are within 5e-5, and within
// 3e-4 where a query's channels differ by factors of a thousand over keys with
// outlier channels; the output's error is the same for all of these.
//   16-bit tokens (sink, window) use the same MMAs on their own type, with ones,
// and bf16 probabilities are split into two parts there.
//
// Work.  The tiles of all (sequence, head) units form one list that is cut
// into equal ranges, one per resident CTA, so ragged lengths balance without
// the host knowing them; the four warps of a CTA take every fourth tile of its
// range, each with a ring of bulk copies of its own (one 4608-byte copy per
// tile) and no synchronisation until a unit ends.  A unit inside one range is
// written at once, the others leave fp32 partials that merge_kernel joins.
//
// What bounds it: 566 warp instructions per tile of 32 tokens (half of them
// bit operations that expand codes, 34 MMAs) against 4608 bytes, at 12 warps
// per SM; issue slots are 59% busy and DRAM at 80% of a copy's rate.  32
// sequences of 32768 tokens, 8 key heads, 1.22 GB: 227 us (5.4 TB/s), 251 to
// 258 us when run back to back, where the board's power limit lowers the
// clocks; one sequence of 4096 tokens: 10.6 us, of which (on an earlier state)
// the list takes 1.2, the first copy 0.7, a tile 2, the join 1 and the merge 2.
// Earlier states: a tile's logits next to the values of the tile before it took
// 224 us to 216; three CTAs of 168 registers with rings of three against four of
// 128 with rings of two (spills) 232 against 228-245 us, and 73 against 84 us on
// 96 sequences of 1 to 20000 tokens.
#include <algorithm>

#include "async_ptx.cuh"
#include "innerq_internal.h"
#include "paged.cuh"

namespace innerq {
namespace {

constexpr int kWarps = 4;
constexpr int kStages = 3;
constexpr int kCtasPerSm = 3;
// what a unit costs beyond its tiles, in tiles: 96 sequences of 1 to 20000
// tokens take 75.7 us with 12, 71.9 with 16, 74.0 with 24 (an earlier state of
// the kernel 277 with 0, 123 with 4); 32 of 32768 do not care (255 us)
constexpr int kUnitCost = 16;
constexpr int kHeadPitch = 148;  // floats per head of the combine buffer: conflict-free
constexpr float kPScale = 8.f;   // probabilities carry 2^8 relative to the running maximum,
constexpr float kSlack = 7.f;    // which may lag behind the true one by 2^7 before it is raised
constexpr float kOutScale = 1048576.f;  // what the values' 2^-20 left in the accumulators
constexpr float kNoMax = -1e30f; // running maximum before the first logit

struct AttnDev {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  uint16_t* out;
  int64_t o_sb, o_sh;
  float* lse;
  float* po;        // [2 grid][R][kD]
  float* pm;        // [2 grid][R]
  float* pl;
  int32_t* starts;  // [B + 1] first place of each sequence in the list
  float scale_log2;
  int Hq, R, cap;   // cap: most tiles a sequence can have
  uint32_t page_bytes;
  int step_page, step_tile;  // kWarps tiles on, in whole pages and tiles
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
// d = a b + c; c stays in its registers, so an accumulator that starts at a
// value used many times costs no moves
template <int DT>
__device__ __forceinline__ void mma_from(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1, const float c[4]) {
  if constexpr (DT == F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// the quad (c0, c1, c0, c1), kept as four registers of its own
__device__ __forceinline__ void quad(float q[4], float c0, float c1) {
  q[0] = q[2] = c0;
  q[1] = q[3] = c1;
  asm("" : "+f"(q[0]), "+f"(q[1]), "+f"(q[2]), "+f"(q[3]));
}
template <int DT>
__device__ __forceinline__ void mma_acc(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  const uint32_t b[2] = {b0, b1};
  mma_dt<DT>(d, a, b);
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// the two halves of a word of the dtype as fp32, one instruction each
template <int DT> __device__ __forceinline__ float lo_f(uint32_t w) {
  if constexpr (DT == F16) return __low2float(*reinterpret_cast<const __half2*>(&w));
  return __uint_as_float(w << 16);
}
template <int DT> __device__ __forceinline__ float hi_f(uint32_t w) {
  if constexpr (DT == F16) return __high2float(*reinterpret_cast<const __half2*>(&w));
  return __uint_as_float(w & 0xffff0000u);
}
// w >> 8, opaque: kept as one shift for both operands taken from it
__device__ __forceinline__ uint32_t shift8(uint32_t w) {
  uint32_t r;
  asm("shr.b32 %0, %1, 8;\n" : "=r"(r) : "r"(w));
  return r;
}

// two code words (rows gid and gid + 8 of an A operand) -> the operands of two
// k-steps: slots 0-7 hold nibbles 0, 4 (2, 6), slots 8-15 nibbles 1, 5 (3, 7)
__device__ __forceinline__ void code_frags(uint32_t w0, uint32_t w1, uint32_t a[4], uint32_t b[4]) {
  a[0] = w0 & 0x000f000fu;
  a[1] = w1 & 0x000f000fu;
  a[2] = w0 & 0x00f000f0u;
  a[3] = w1 & 0x00f000f0u;
  w0 = shift8(w0);
  w1 = shift8(w1);
  b[0] = w0 & 0x000f000fu;
  b[1] = w1 & 0x000f000fu;
  b[2] = w0 & 0x00f000f0u;
  b[3] = w1 & 0x00f000f0u;
}

// The same slots with every code four bits up, u 2^-20.
__device__ __forceinline__ void value_frags(uint32_t w0, uint32_t w1, uint32_t a[4], uint32_t b[4]) {
  a[0] = (w0 << 4) & 0x00f000f0u;
  a[1] = (w1 << 4) & 0x00f000f0u;
  a[2] = w0 & 0x00f000f0u;
  a[3] = w1 & 0x00f000f0u;
  b[0] = (w0 >> 4) & 0x00f000f0u;
  b[1] = (w1 >> 4) & 0x00f000f0u;
  b[2] = (w0 >> 8) & 0x00f000f0u;
  b[3] = (w1 >> 8) & 0x00f000f0u;
}

// What one warp has accumulated of a unit.  A lane holds the query heads
// 2 tq + {0, 1} and, of each, the channels 16 gid + 2 mt + {0, 1}:
// acc[mt][2 i + c] is channel 16 gid + 2 mt + i of head 2 tq + c; acc and l carry
// 2^8.
struct State {
  float acc[8][4], m[2], l[2];
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    m[0] = m[1] = kNoMax;
    l[0] = l[1] = 0.f;
  }
  __device__ __forceinline__ void poison() {
    l[0] = l[1] = NAN;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = NAN;
  }
  // this lane's largest logits of a tile x[row pair][..] f (f >= 0) per column
  __device__ __forceinline__ void largest(const float x[2][4], float f0, float f1, float& t0, float& t1) const {
    t0 = fmaxf(fmaxf(x[0][0], x[0][2]), fmaxf(x[1][0], x[1][2])) * f0;
    t1 = fmaxf(fmaxf(x[0][1], x[0][3]), fmaxf(x[1][1], x[1][3])) * f1;
  }
  // No lane's logits lie more than the slack above the running maximum.  The
  // maximum over the lanes is only taken where this fails.
  __device__ __forceinline__ bool fits(float t0, float t1) const {
    return !__any_sync(~0u, t0 > m[0] + kSlack || t1 > m[1] + kSlack);
  }
  // raise the running maxima and rescale
  __device__ __forceinline__ void raise(float t0, float t1) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      t0 = fmaxf(t0, __shfl_xor_sync(~0u, t0, o));
      t1 = fmaxf(t1, __shfl_xor_sync(~0u, t1, o));
    }
    const float n0 = fmaxf(m[0], t0), n1 = fmaxf(m[1], t1), c0 = ex2(m[0] - n0), c1 = ex2(m[1] - n1);
    m[0] = n0;
    m[1] = n1;
    l[0] *= c0;
    l[1] *= c1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      acc[i][0] *= c0;
      acc[i][1] *= c1;
      acc[i][2] *= c0;
      acc[i][3] *= c1;
    }
  }
};

// The query of a unit as MMA operands: lane (gid, tq) holds head gid's
// channels 32 g + 8 tq + 0..7 as B operands, and for its columns (heads
// 2 tq + {0, 1}) the offset terms and the factor of the logits.
struct Query {
  uint32_t b[16];
  float off[4][4];
  float f[2];
};

template <int DT>
__device__ __forceinline__ void load_query(const AttnDev& a, int b, int h, int lane, Query& o) {
  const int gid = lane >> 2, tq = lane & 3;
  uint4 w[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) w[g] = make_uint4(0, 0, 0, 0);
  if (gid < a.R) {
    const uint4* src = reinterpret_cast<const uint4*>(a.q + b * a.q_sb + (int64_t)(h * a.R + gid) * a.q_sh) + tq;
#pragma unroll
    for (int g = 0; g < 4; ++g) w[g] = __ldg(src + 4 * g);
  }
  float top = 0.f;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const uint32_t* x = reinterpret_cast<const uint32_t*>(&w[g]);
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(lo_f<DT>(x[i])), fabsf(hi_f<DT>(x[i]))));
  }
  top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
  top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
  int e = 0;
  if (top > 0.f && top < INFINITY) e = min(100, max(-100, 14 - ilogbf(top)));
  // the sign of the softmax scale goes into q, so that f >= 0 and the largest
  // raw product is the largest logit
  const float up = a.scale_log2 < 0.f ? -exp2f((float)e) : exp2f((float)e);
  float sum[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const uint32_t* x = reinterpret_cast<const uint32_t*>(&w[g]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = lo_f<DT>(x[i]) * up;
      v[2 * i + 1] = hi_f<DT>(x[i]) * up;
    }
    sum[g] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    sum[g] += __shfl_xor_sync(~0u, sum[g], 1);
    sum[g] += __shfl_xor_sync(~0u, sum[g], 2);
    o.b[4 * g] = half2_of(v[0], v[4]);
    o.b[4 * g + 1] = half2_of(v[1] * 0.0625f, v[5] * 0.0625f);
    o.b[4 * g + 2] = half2_of(v[2], v[6]);
    o.b[4 * g + 3] = half2_of(v[3] * 0.0625f, v[7] * 0.0625f);
  }
  const float f = fabsf(a.scale_log2) * exp2f((float)(24 - e));
  o.f[0] = __shfl_sync(~0u, f, 8 * tq);
  o.f[1] = __shfl_sync(~0u, f, 8 * tq + 4);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const float s0 = __shfl_sync(~0u, sum[g], 8 * tq), s1 = __shfl_sync(~0u, sum[g], 8 * tq + 4);
    quad(o.off[g], s0 * (-8.f / 16777216.f), s1 * (-8.f / 16777216.f));
  }
}

// logits of a packed tile in shared memory, before the factor q.f
template <int DT>
__device__ __forceinline__ void packed_logits(const uint8_t* blk, int lane, const Query& q, float x[2][4]) {
  const int gid = lane >> 2;
#pragma unroll
  for (int mm = 0; mm < 2; ++mm) {
    const uint4 w0 = reinterpret_cast<const uint4*>(blk)[64 * mm + lane];
    const uint4 w1 = reinterpret_cast<const uint4*>(blk)[64 * mm + 32 + lane];
    // scales of rows 8 (2 mm) + gid and 8 (2 mm + 1) + gid, four groups each
    const uint4 sc = reinterpret_cast<const uint4*>(blk + kKScale)[2 * gid + mm];
    const uint32_t* p0 = reinterpret_cast<const uint32_t*>(&w0);
    const uint32_t* p1 = reinterpret_cast<const uint32_t*>(&w1);
    const uint32_t* ps = reinterpret_cast<const uint32_t*>(&sc);
    x[mm][0] = x[mm][1] = x[mm][2] = x[mm][3] = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t a[4], b[4];
      code_frags(p0[g], p1[g], a, b);
      float d[4];
      mma_from<F16>(d, a, q.b[4 * g], q.b[4 * g + 1], q.off[g]);
      mma_acc<F16>(d, b, q.b[4 * g + 2], q.b[4 * g + 3]);
      const float s0 = g & 1 ? hi_f<DT>(ps[g >> 1]) : lo_f<DT>(ps[g >> 1]);
      const float s1 = g & 1 ? hi_f<DT>(ps[2 + (g >> 1)]) : lo_f<DT>(ps[2 + (g >> 1)]);
      x[mm][0] = fmaf(s0, d[0], x[mm][0]);
      x[mm][1] = fmaf(s0, d[1], x[mm][1]);
      x[mm][2] = fmaf(s1, d[2], x[mm][2]);
      x[mm][3] = fmaf(s1, d[3], x[mm][3]);
    }
  }
}

// its probabilities and values
template <int DT>
__device__ __forceinline__ void packed_values(const uint8_t* blk, int lane, const Query& q, const float x[2][4], State& s) {
  const int gid = lane >> 2;
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  const float b0 = kPScale - s.m[0], b1 = kPScale - s.m[1];
  uint32_t pb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    pb[i] = transpose8x8(half2_of(ex2(fmaf(x[i >> 1][2 * (i & 1)], q.f[0], b0)), ex2(fmaf(x[i >> 1][2 * (i & 1) + 1], q.f[1], b1))));
  float ps[4];
  // 8 sum p, the offset; an eighth of it divides the result
  const uint32_t eights[4] = {0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u};
  mma_from<F16>(ps, eights, pb[0], pb[1], zero);
  mma_acc<F16>(ps, eights, pb[2], pb[3]);
  s.l[0] = fmaf(ps[0], kOutScale / 8.f, s.l[0]);
  s.l[1] = fmaf(ps[1], kOutScale / 8.f, s.l[1]);
  float off[4];
  quad(off, -ps[0], -ps[1]);
  const uint4 v0 = reinterpret_cast<const uint4*>(blk + kVScale)[2 * gid];
  const uint4 v1 = reinterpret_cast<const uint4*>(blk + kVScale)[2 * gid + 1];
#pragma unroll
  for (int pc = 0; pc < 4; ++pc) {
    const uint4 w = reinterpret_cast<const uint4*>(blk + kVCodes)[32 * pc + lane];
    const uint32_t* pw = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int mt = 2 * pc + m;
      uint32_t a[4], b[4];
      value_frags(pw[2 * m], pw[2 * m + 1], a, b);
      float d[4];
      mma_from<F16>(d, a, pb[0], pb[1], off);
      mma_acc<F16>(d, b, pb[2], pb[3]);
      const uint32_t sc = reinterpret_cast<const uint32_t*>(mt < 4 ? &v0 : &v1)[mt & 3];
      const float s0 = lo_f<DT>(sc), s1 = hi_f<DT>(sc);
      s.acc[mt][0] = fmaf(s0, d[0], s.acc[mt][0]);
      s.acc[mt][1] = fmaf(s0, d[1], s.acc[mt][1]);
      s.acc[mt][2] = fmaf(s1, d[2], s.acc[mt][2]);
      s.acc[mt][3] = fmaf(s1, d[3], s.acc[mt][3]);
    }
  }
}

template <int DT> __device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  return w & ((not_finite<DT>(w) ? 0u : 0xffffu) | (not_finite<DT>(w >> 16) ? 0u : 0xffff0000u));
}

// one 16-bit tile (sink or window) straight from global memory: kr / vr point
// at its first row, `valid` of its 32 rows hold tokens.  An infinite value counts
// with any probability above 0, of which an fp16 operand may be 0 and a second
// part 0 or negative: `seen` becomes NaN where a sum is not finite, and the
// unit's tiles are then taken again with ONE_BY_ONE, which adds the values that
// are not finite in fp32.
template <int DT, bool ONE_BY_ONE>
__device__ __forceinline__ void dense_tile(const uint16_t* kr, const uint16_t* vr, int valid, const AttnDev& a, int b, int h,
                                        int lane, float& seen, State& s) {
  const int gid = lane >> 2, tq = lane & 3;
  uint4 qw[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) qw[g] = make_uint4(0, 0, 0, 0);
  if (gid < a.R) {
    const uint4* src = reinterpret_cast<const uint4*>(a.q + b * a.q_sb + (int64_t)(h * a.R + gid) * a.q_sh) + tq;
#pragma unroll
    for (int g = 0; g < 4; ++g) qw[g] = __ldg(src + 4 * g);
  }
  float x[2][4];
#pragma unroll
  for (int mm = 0; mm < 2; ++mm) {
    const uint4* r0 = reinterpret_cast<const uint4*>(kr + (16 * mm + gid) * kD) + tq;
    const uint4* r1 = r0 + 8 * kD / 8;
    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint4 y0 = r0[4 * g], y1 = r1[4 * g];
      const uint32_t a0[4] = {y0.x, y1.x, y0.y, y1.y}, a1[4] = {y0.z, y1.z, y0.w, y1.w};
      mma_acc<DT>(d, a0, qw[g].x, qw[g].y);
      mma_acc<DT>(d, a1, qw[g].z, qw[g].w);
    }
    const bool in0 = 16 * mm + gid < valid, in1 = 16 * mm + 8 + gid < valid;
    x[mm][0] = in0 ? d[0] * a.scale_log2 : -INFINITY;
    x[mm][1] = in0 ? d[1] * a.scale_log2 : -INFINITY;
    x[mm][2] = in1 ? d[2] * a.scale_log2 : -INFINITY;
    x[mm][3] = in1 ? d[3] * a.scale_log2 : -INFINITY;
  }
  float t0, t1;
  s.largest(x, 1.f, 1.f, t0, t1);
  if (!s.fits(t0, t1)) s.raise(t0, t1);
  uint32_t pb[4], pe[4];  // bf16: the rounded probabilities and what the rounding left
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float p0 = ex2(x[i >> 1][2 * (i & 1)] - s.m[0] + kPScale), p1 = ex2(x[i >> 1][2 * (i & 1) + 1] - s.m[1] + kPScale);
    const uint16_t h0 = from_f<DT>(p0), h1 = from_f<DT>(p1);
    pb[i] = transpose8x8(pack2(h0, h1));
    if constexpr (DT == BF16) pe[i] = transpose8x8(pack2(from_f<DT>(p0 - to_f<DT>(h0)), from_f<DT>(p1 - to_f<DT>(h1))));
  }
  float ps[4];
  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  const uint32_t one = DT == F16 ? 0x3c003c00u : 0x3f803f80u;
  const uint32_t ones[4] = {one, one, one, one};
  mma_from<DT>(ps, ones, pb[0], pb[1], zero);
  mma_acc<DT>(ps, ones, pb[2], pb[3]);
  if constexpr (DT == BF16) {
    mma_acc<DT>(ps, ones, pe[0], pe[1]);
    mma_acc<DT>(ps, ones, pe[2], pe[3]);
  }
  s.l[0] += ps[0];
  s.l[1] += ps[1];
#pragma unroll
  for (int part = 0; part < 4; ++part) {  // channels 16 gid + 4 part ..: m-tiles 2 part, 2 part + 1
    uint2 v[8];                           // tokens 2 tq + {0, 1, 8, 9, 16, 17, 24, 25}
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = 8 * (i >> 1) + 2 * tq + (i & 1);
      v[i] = reinterpret_cast<const uint2*>(vr + t * kD)[4 * gid + part];
      if (t >= valid) v[i] = make_uint2(0, 0);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = m ? v[i].y : v[i].x;
      if constexpr (ONE_BY_ONE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = finite_halves<DT>(w[i]);
      }
      uint32_t f[2][4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f[k][0] = __byte_perm(w[4 * k], w[4 * k + 1], 0x5410);
        f[k][1] = __byte_perm(w[4 * k], w[4 * k + 1], 0x7632);
        f[k][2] = __byte_perm(w[4 * k + 2], w[4 * k + 3], 0x5410);
        f[k][3] = __byte_perm(w[4 * k + 2], w[4 * k + 3], 0x7632);
      }
      float d[4];
      mma_from<DT>(d, f[0], pb[0], pb[1], zero);
      mma_acc<DT>(d, f[1], pb[2], pb[3]);
      if constexpr (DT == BF16) {
        mma_acc<DT>(d, f[0], pe[0], pe[1]);
        mma_acc<DT>(d, f[1], pe[2], pe[3]);
      }
      if constexpr (ONE_BY_ONE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = ex2(x[i >> 1][2 * (i & 1)] - s.m[0] + kPScale), p1 = ex2(x[i >> 1][2 * (i & 1) + 1] - s.m[1] + kPScale);
#pragma unroll 1
          for (int j = 0; j < 8; ++j) {  // token 8 i + j: its probabilities are with lanes 4 j ..
            const float y0 = __shfl_sync(~0u, p0, 4 * j + tq), y1 = __shfl_sync(~0u, p1, 4 * j + tq);
            if (8 * i + j >= valid) continue;
            const uint32_t y = reinterpret_cast<const uint32_t*>(vr + (8 * i + j) * kD)[8 * gid + 2 * part + m];
            if (not_finite<DT>(y)) d[0] = fmaf(y0, lo_f<DT>(y), d[0]), d[1] = fmaf(y1, lo_f<DT>(y), d[1]);
            if (not_finite<DT>(y >> 16)) d[2] = fmaf(y0, hi_f<DT>(y), d[2]), d[3] = fmaf(y1, hi_f<DT>(y), d[3]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) seen = fmaf(d[i], 0.f, seen);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s.acc[2 * part + m][i] = fmaf(d[i], 1.f / kOutScale, s.acc[2 * part + m][i]);
    }
  }
}

// a warp's 16-bit tiles of a unit that begins at place u0: every fourth place from
// idx to end but the packed ones.  True: some sum is not finite.
template <int DT, bool ONE_BY_ONE>
__device__ __forceinline__ bool dense_tiles(const PagedDev& c, const AttnDev& a, int b, int h, int u0, int idx, int packed_lo,
                                            int packed_end, int end, int lane, State& s) {
  float seen = 0.f;
  s.reset();
#pragma unroll 1
  for (int p = idx;; p += kWarps) {
    if (p >= packed_lo && p < packed_end) p = packed_end + ((p - packed_end) & (kWarps - 1));
    if (p >= end) break;
    const int64_t base = c.dense_base(b, h);
    if (base < 0) {
      s.poison();
      continue;
    }
    const int t = 32 * (p - u0);
    const int64_t at = base + (int64_t)c.row_of(t) * kD;
    dense_tile<DT, ONE_BY_ONE>(c.dk + at, c.dv + at, c.lens[b] - t, a, b, h, lane, seen, s);
  }
  return __any_sync(~0u, seen != 0.f);
}
template <int DT>
__device__ __noinline__ void dense_tiles_one_by_one(const PagedDev& c, const AttnDev& a, int b, int h, int u0, int idx, int packed_lo,
                                                    int packed_end, int end, int lane, State* s) {
  dense_tiles<DT, true>(c, a, b, h, u0, idx, packed_lo, packed_end, end, lane, *s);
}

__device__ __forceinline__ int tiles_in(int len, int cap) { return len <= 0 ? 0 : min((int)(((int64_t)len + 31) >> 5), cap); }
__device__ __forceinline__ int tiles_of(const PagedDev& c, int b, int cap) { return tiles_in(c.lens[b], cap); }

// length of a unit of nt tiles in the list: a unit takes time beyond its tiles
// (its query, its first loads, the join), so it is followed by kUnitCost
// places that hold no tile
__device__ __forceinline__ int places_of(int nt) { return nt ? nt + kUnitCost : 0; }

__device__ __forceinline__ int warp_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(~0u, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

template <int RH>
struct alignas(128) Smem {
  uint8_t ring[kWarps][kStages][kBlockBytes];
  float buf[2][RH][kHeadPitch];
  float m[kWarps][8], l[kWarps][8];
  uint64_t bars[kWarps][kStages];
  int4 put[kWarps];
  int bad[kWarps];
};

// tiles per CTA: equal ranges, whole rounds of the four warps
__device__ __forceinline__ int range_of(int total, int grid) {
  return max(kWarps, ((total + grid - 1) / grid + kWarps - 1) / kWarps * kWarps);
}

template <int DT, int RH>
__global__ void __launch_bounds__(128, kCtasPerSm) attn_kernel(const __grid_constant__ PagedDev c, const __grid_constant__ AttnDev a) {
  extern __shared__ __align__(128) uint8_t raw[];
  Smem<RH>& sm = *reinterpret_cast<Smem<RH>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) mbar_init(&sm.bars[w][i], 1);
    mbar_fence_init();
  }
  griddep_wait();
  griddep_launch_dependents();

  // the list of tiles: where this CTA's range begins (every warp for itself)
  auto length = [&](int b) { return b < c.B ? c.lens[b] : 0; };
  auto places = [&](int len) { return places_of(tiles_in(len, a.cap)) * c.Hkv; };
  int total = 0;
  for (int b0 = 0; b0 < c.B; b0 += 32) total += __reduce_add_sync(~0u, places(length(b0 + lane)));
  const int per = range_of(total, gridDim.x);
  const int lo = blockIdx.x * per, hi = min(total, lo + per);
  if (blockIdx.x == 0 && w == 0) {  // for merge_kernel
    for (int b0 = 0, at = 0; b0 < c.B; b0 += 32) {
      const int v = places(length(b0 + lane)), end = at + warp_scan(v, lane);
      if (b0 + lane < c.B) a.starts[b0 + lane] = end - v;
      at = __shfl_sync(~0u, end, 31);
    }
    if (lane == 0) a.starts[c.B] = total;
  }
  if (lo >= total) return;
  int b = 0, nt = 0, u0 = 0, packed = 0;
  for (int b0 = 0, at = 0;; b0 += 32) {
    const int len = length(b0 + lane), v = places(len), sum = __reduce_add_sync(~0u, v);
    if (lo < at + sum) {
      const int end = at + warp_scan(v, lane);
      const int src = __ffs(__ballot_sync(~0u, lo < end)) - 1;
      b = b0 + src;
      u0 = __shfl_sync(~0u, end - v, src);
      const int l = __shfl_sync(~0u, len, src);
      nt = tiles_in(l, a.cap);
      packed = c.n_packed(l) >> 5;
      break;
    }
    at += sum;
  }
  int h = (lo - u0) / places_of(nt);
  u0 += h * places_of(nt);
  const int sink_tiles = c.w_sink >> 5;
  // the unit after (b, h); false when it begins outside the range
  auto advance = [&]() {
    u0 += places_of(nt);
    if (u0 >= hi) return false;
    if (++h == c.Hkv) {
      h = 0;
      do {
        ++b;
        nt = tiles_of(c, b, a.cap);
      } while (nt == 0);
      packed = c.n_packed(c.lens[b]) >> 5;
    }
    return true;
  };
  if (lo >= u0 + nt && !advance()) return;

  // The unit's tiles of this CTA are the places [max(lo, u0), min(hi, u0 + nt))
  // of the list; of those this warp takes every fourth, the packed ones through
  // its ring.  Lane 0 keeps the copies ahead; the page number of its next copy
  // is loaded one tile early, so that no tile waits for the table.
  int idx = max(lo, u0) + w;
  int in_flight = 0;             // copies under way (lane 0)
  int st_put = 0, st_get = 0;    // ring slots of the next copy and the next tile
  uint32_t parity = 0;
  // in shared memory: copies of this unit not yet issued, the next one's page,
  // tile in the page and page number
  int4& put = sm.put[w];
  auto page_number = [&](int left, int page) {
    return left > 0 && page < c.max_pages ? c.table[b * c.table_stride + page] : -1;
  };
  auto issue = [&]() {
    int4 p = put;
    if (p.x <= 0) return;
    if ((unsigned)p.w < (unsigned)c.n_pages) {
      mbar_arrive_tx(&sm.bars[w][st_put], kBlockBytes);
      bulk_g2s(sm.ring[w][st_put],
               c.pages + (uint64_t)a.page_bytes * (uint32_t)p.w + (uint32_t)((h * c.page_tiles + p.z) * kBlockBytes),
               kBlockBytes, &sm.bars[w][st_put]);
    } else {  // no such page: whatever the slot holds is used and the unit becomes NaN
      sm.bad[w] = 1;
      mbar_arrive(&sm.bars[w][st_put]);
    }
    if (++st_put == kStages) st_put = 0;
    ++in_flight;
    --p.x;
    p.y += a.step_page;
    p.z += a.step_tile;
    if (p.z >= c.page_tiles) {
      p.z -= c.page_tiles;
      ++p.y;
    }
    p.w = page_number(p.x, p.y);
    put = p;
  };
  auto begin_unit = [&]() {
    if (lane) return;
    const int first = max(idx, u0 + sink_tiles + ((idx - u0 - sink_tiles) & (kWarps - 1)));
    const int left = (min(hi, u0 + sink_tiles + packed) - first + kWarps - 1) >> 2;
    const int t = max(0, first - u0 - sink_tiles), page = t / c.page_tiles;
    put = make_int4(left, page, t - page * c.page_tiles, page_number(left, page));
#pragma unroll
    for (int i = 0; i < kStages; ++i) issue();
  };
  sm.bad[w] = 0;
  __syncwarp();
  begin_unit();

  bool failed = false;
  State s;
  while (true) {
    const int end = min(hi, u0 + nt);
    // the 16-bit tiles (sink and window) first, while the copies are under way
    const int packed_lo = u0 + sink_tiles, packed_end = min(end, packed_lo + packed);
    if (dense_tiles<DT, false>(c, a, b, h, u0, idx, packed_lo, packed_end, end, lane, s)) {
      State again;
      dense_tiles_one_by_one<DT>(c, a, b, h, u0, idx, packed_lo, packed_end, end, lane, &again);
      s = again;
    }
    if (idx < packed_lo) idx = packed_lo + ((idx - packed_lo) & (kWarps - 1));
    if (idx < packed_end) {
      Query q;
      load_query<DT>(a, b, h, lane, q);
      // The logits of a tile are computed next to the values of the one before
      // it: two independent streams of instructions.
      float x[2][4];
      auto logits = [&](int st, float y[2][4]) { packed_logits<DT>(sm.ring[w][st], lane, q, y); };
      auto settle = [&]() {
        float t0, t1;
        s.largest(x, q.f[0], q.f[1], t0, t1);
        if (!s.fits(t0, t1)) s.raise(t0, t1);
      };
      failed = failed || !mbar_wait_warp(&sm.bars[w][st_get], parity, kWaitLimit);
      if (!failed) {
        logits(st_get, x);
        settle();
      }
#pragma unroll 1
      while (!failed) {
        const int st = st_get;
        if (++st_get == kStages) {
          st_get = 0;
          parity ^= 1;
        }
        idx += kWarps;
        if (idx >= packed_end) {
          packed_values<DT>(sm.ring[w][st], lane, q, x, s);
          __syncwarp();
          if (lane == 0) --in_flight;
          break;
        }
        failed = !mbar_wait_warp(&sm.bars[w][st_get], parity, kWaitLimit);
        if (failed) break;
        float y[2][4];
        packed_values<DT>(sm.ring[w][st], lane, q, x, s);
        logits(st_get, y);
        __syncwarp();
        if (lane == 0) {
          --in_flight;
          issue();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) x[0][i] = y[0][i], x[1][i] = y[1][i];
        settle();
      }
      if (failed) s.poison();
    }
    // the next unit's copies go out before this one is joined
    const bool whole = lo <= u0 && u0 + nt <= hi;
    const int slot = 2 * blockIdx.x + (lo > u0 ? 0 : 1), ob = b, oh = h;
    const bool bad = sm.bad[w];
    __syncwarp();
    if (bad) {
      s.poison();
      if (lane == 0) sm.bad[w] = 0;
    }
    const bool more = advance();
    if (more) {
      idx = u0 + w;
      if (!failed) begin_unit();
    }
    // join the four warps
    const int gid = lane >> 2, tq = lane & 3;
    if (gid == 0) {
      sm.m[w][2 * tq] = s.m[0];
      sm.m[w][2 * tq + 1] = s.m[1];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float top =
          fmaxf(fmaxf(sm.m[0][2 * tq + i], sm.m[1][2 * tq + i]), fmaxf(sm.m[2][2 * tq + i], sm.m[3][2 * tq + i]));
      const float f = ex2(s.m[i] - top);
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        s.acc[mt][i] *= f;
        s.acc[mt][i + 2] *= f;
      }
      if (gid == 0) sm.l[w][2 * tq + i] = s.l[i] * f;
    }
    // warps 2 and 3 hand over to 0 and 1, which leave two sums
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
      if ((w < 2) == (turn == 1)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (2 * tq + i < RH) {
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) {
              float2* at = reinterpret_cast<float2*>(&sm.buf[w & 1][2 * tq + i][18 * gid + 2 * mt]);
              const float2 add = turn ? *at : make_float2(0.f, 0.f);
              *at = make_float2(s.acc[mt][i] + add.x, s.acc[mt][i + 2] + add.y);
            }
          }
        }
      }
      __syncthreads();
    }
    for (int r = 0; r < a.R; ++r) {
      const int at = 18 * (tid >> 4) + (tid & 15);
      const float o = sm.buf[0][r][at] + sm.buf[1][r][at];
      const float l = (sm.l[0][r] + sm.l[1][r]) + (sm.l[2][r] + sm.l[3][r]);
      const float m = fmaxf(fmaxf(sm.m[0][r], sm.m[1][r]), fmaxf(sm.m[2][r], sm.m[3][r]));
      if (whole) {
        const int hq = oh * a.R + r;
        a.out[ob * a.o_sb + hq * a.o_sh + tid] = from_f<DT>(o * kOutScale / l);
        if (a.lse && tid == 0) a.lse[(int64_t)ob * a.Hq + hq] = m + log2f(l) - kPScale;
      } else {
        a.po[((int64_t)slot * a.R + r) * kD + tid] = o;
        if (tid == 0) {
          a.pm[slot * a.R + r] = m;
          a.pl[slot * a.R + r] = l;
        }
      }
    }
    if (!more) break;
    __syncthreads();
  }
  if (failed && lane == 0) {  // copies still in flight must land before the CTA's memory is given away
    for (; in_flight > 0; --in_flight) {
      mbar_wait_bounded(&sm.bars[w][st_get], parity, kWaitLimit / 16);
      if (++st_get == kStages) {
        st_get = 0;
        parity ^= 1;
      }
    }
  }
}

// Joins the partials of the units that were cut; zeros for units without
// tokens.  One block per (head, sequence): its warps take the partials in
// turn, four at a time so that their loads overlap, then join.
constexpr int kMergeWarps = 8;
template <int DT>
__global__ void __launch_bounds__(32 * kMergeWarps) merge_kernel(AttnDev a, int Hkv, int grid, int B) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ float4 so[kMergeWarps][32];
  __shared__ float sm[kMergeWarps], sl[kMergeWarps];
  const int b = blockIdx.y, hq = blockIdx.x, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int s0 = a.starts[b], places = (a.starts[b + 1] - s0) / Hkv, nt = places - kUnitCost;
  uint16_t* out = a.out + b * a.o_sb + hq * a.o_sh;
  if (places == 0) {
    if (threadIdx.x < kD) out[threadIdx.x] = 0;
    if (a.lse && threadIdx.x == 0) a.lse[(int64_t)b * a.Hq + hq] = -INFINITY;
    return;
  }
  const int per = range_of(a.starts[B], grid);
  const int u0 = s0 + hq / a.R * places, r = hq % a.R;
  const int c0 = u0 / per, c1 = (u0 + nt - 1) / per;
  if (c0 == c1) return;
  float m = kNoMax, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto join = [&](float pm, float pl, float4 po) {
    const float n = fmaxf(m, pm), f = ex2(m - n), g = ex2(pm - n);
    m = n;
    l = l * f + pl * g;
    o.x = o.x * f + po.x * g;
    o.y = o.y * f + po.y * g;
    o.z = o.z * f + po.z * g;
    o.w = o.w * f + po.w * g;
  };
  for (int i0 = c0 + w; i0 <= c1; i0 += 4 * kMergeWarps) {
    float pm[4], pl[4];
    float4 po[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * kMergeWarps;
      pm[j] = kNoMax;
      pl[j] = 0.f;
      po[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i <= c1) {
        const int64_t s = (int64_t)(2 * i + (i * per > u0 ? 0 : 1)) * a.R + r;
        pm[j] = a.pm[s];
        pl[j] = a.pl[s];
        po[j] = reinterpret_cast<const float4*>(a.po + s * kD)[lane];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) join(pm[j], pl[j], po[j]);
  }
  so[w][lane] = o;
  if (lane == 0) {
    sm[w] = m;
    sl[w] = l;
  }
  __syncthreads();
  if (w) return;
#pragma unroll
  for (int i = 1; i < kMergeWarps; ++i) join(sm[i], sl[i], so[i][lane]);
  const float inv = kOutScale / l;
  uint16_t* at = out + 4 * lane;
  at[0] = from_f<DT>(o.x * inv);
  at[1] = from_f<DT>(o.y * inv);
  at[2] = from_f<DT>(o.z * inv);
  at[3] = from_f<DT>(o.w * inv);
  if (a.lse && lane == 0) a.lse[(int64_t)b * a.Hq + hq] = m + log2f(l) - kPScale;
}

int grid_size() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148 * kCtasPerSm;
  if (!cached[dev]) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    cached[dev] = (n > 0 ? n : 148) * kCtasPerSm;
  }
  return cached[dev];
}

template <int DT, int RH>
cudaError_t launch_attn(const PagedDev& c, const AttnDev& a, int grid, cudaStream_t s) {
  static bool ready[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !ready[dev]) {
    e = cudaFuncSetAttribute(attn_kernel<DT, RH>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem<RH>));
    if (e != cudaSuccess) return e;
    if (dev < 64) ready[dev] = true;
  }
  e = launch_pdl(attn_kernel<DT, RH>, dim3(grid), dim3(128), sizeof(Smem<RH>), s, c, a);
  if (e != cudaSuccess) return e;
  return launch_pdl(merge_kernel<DT>, dim3(a.Hq, c.B), dim3(32 * kMergeWarps), 0, s, a, c.Hkv, grid, c.B);
}

int64_t workspace_bytes_of(int grid, int R, int B) {
  return (int64_t)2 * grid * R * (kD + 2) * 4 + ((int64_t)B + 1) * 4 + 256;
}

int check_heads(const PagedDev& c, int Hq) {
  if (Hq <= 0 || Hq % c.Hkv) return set_last_error(INNERQ_ERR_ARG, "%d query heads over %d key heads", Hq, c.Hkv);
  if (Hq / c.Hkv > 8) return set_last_error(INNERQ_ERR_UNSUPPORTED, "GQA ratio %d (1 to 8 are built)", Hq / c.Hkv);
  return INNERQ_OK;
}

}  // namespace
}  // namespace innerq

using namespace innerq;

extern "C" int64_t innerq_paged_attn_workspace(const innerq_paged* cache, int Hq) {
  PagedDev c;
  if (paged_dev(cache, c) || check_heads(c, Hq)) return -1;
  return workspace_bytes_of(grid_size(), Hq / c.Hkv, c.B);
}

extern "C" int innerq_paged_attn(const innerq_paged* cache, int Hq, const void* q, int64_t q_sb, int64_t q_sh, float scale,
                                 void* workspace, int64_t workspace_bytes, void* out, int64_t o_sb, int64_t o_sh,
                                 float* lse, void* stream) {
  PagedDev c;
  if (int rc = paged_dev(cache, c)) return rc;
  if (int rc = check_heads(c, Hq)) return rc;
  if (c.B == 0) return INNERQ_OK;
  if (!q || !out || !workspace) return set_last_error(INNERQ_ERR_ARG, "null pointer");
  if (((uintptr_t)q & 15) || ((uintptr_t)workspace & 15) || ((uintptr_t)out & 1) || q_sb % 8 || q_sh % 8)
    return set_last_error(INNERQ_ERR_ARG, "query rows and workspace must be 16-byte aligned");
  if (c.B > 65535) return set_last_error(INNERQ_ERR_ARG, "more than 65535 sequences");
  const int64_t cap = (c.w_sink + c.w_recent) / 32 + 1 + (int64_t)c.max_pages * c.page_tiles;
  if ((int64_t)c.Hkv * c.page_tiles * kBlockBytes > 0xffffffffll) return set_last_error(INNERQ_ERR_ARG, "pages of 4 GiB or more");
  if ((cap + kUnitCost) * c.B * c.Hkv > 0x7fffffffll - (1 << 20))
    return set_last_error(INNERQ_ERR_ARG, "page table of %d x %d is too large for one launch", c.B, c.max_pages);
  const int grid = grid_size(), R = Hq / c.Hkv;
  if (workspace_bytes < workspace_bytes_of(grid, R, c.B))
    return set_last_error(INNERQ_ERR_ARG, "workspace %lld bytes < %lld", (long long)workspace_bytes,
                          (long long)workspace_bytes_of(grid, R, c.B));
  AttnDev a;
  a.q = (const uint16_t*)q;
  a.q_sb = q_sb; a.q_sh = q_sh;
  a.out = (uint16_t*)out;
  a.o_sb = o_sb; a.o_sh = o_sh;
  a.lse = lse;
  a.po = (float*)workspace;
  a.pm = a.po + (int64_t)2 * grid * R * kD;
  a.pl = a.pm + (int64_t)2 * grid * R;
  a.starts = (int32_t*)(a.pl + (int64_t)2 * grid * R);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.Hq = Hq; a.R = R; a.cap = (int)cap;
  a.page_bytes = (uint32_t)c.Hkv * c.page_tiles * kBlockBytes;
  a.step_page = kWarps / c.page_tiles;
  a.step_tile = kWarps % c.page_tiles;
  const cudaStream_t s = (cudaStream_t)stream;
  const bool bf = cache->dtype == INNERQ_DT_BF16;
  const cudaError_t e = R <= 4 ? (bf ? launch_attn<BF16, 4>(c, a, grid, s) : launch_attn<F16, 4>(c, a, grid, s))
                               : (bf ? launch_attn<BF16, 8>(c, a, grid, s) : launch_attn<F16, 8>(c, a, grid, s));
  return e == cudaSuccess ? INNERQ_OK : set_last_error(INNERQ_ERR_CUDA, "paged_attn: %s", cudaGetErrorString(e));
}
