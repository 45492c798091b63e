// Attention of whole prompts packed one behind the other, on the tensor cores
// (tcgen05).
//
// Mathematics.  One pass over key tiles of 128: S = Q K^T, running row
// maximum m and sum l, P = 2^(S scale log2 e - m), O += P V.  m may lag behind
// the true maximum by 2^8 before O is rescaled, so rescaling is rare; P carries
// 2^7 so that fp16 keeps 11 bits down to 2^-21 of the largest.  P is rounded to
// the inputs' type for the second product (its sum l is not); everything else
// is fp32.
//
// A piece of work is two query tiles of 128 rows, a row being one token's query
// of one of the heads that share their keys; one tile's softmax runs while the
// tensor core works for the other:
//   warps 0-3, 4-7  softmax of tile 0 and 1, one thread per query row (no
//                   shuffles); rescaling and the epilogue too
//   warp 8          issues every MMA: S_i = Q_i K^T from shared memory, then
//                   O_i += P_i V with P_i read from tensor memory, where it
//                   replaces S_i
//   warp 9          TMA loads: Q, and K and V tiles through a ring
//   warps 10, 11    look over the V tiles that some row must not see whole: a
//                   masked probability is 0, but 0 * NaN is NaN, so values
//                   that are not finite are set to 0 there and added again, in
//                   the epilogue, to the rows that do see them (as are, in
//                   fp16, those that met a probability below what fp16 holds)
// A CTA stays and takes over blocks that have not started (the grid is one block
// per pair of query tiles and head, heavy ones first), so the loads and scores
// of the next piece of work run under the epilogue of the last; warp 11 asks.
// What bounds it: per key tile of a pair the four products take 2048 cycles of
// the tensor core at least, the exponentials about as many of the special
// function units, and a tile's chain (scores, softmax, P V) some 3200, 2000 of
// them softmax; two tiles overlap it to 58% tensor occupancy (special functions
// 45%, issue slots 47%), and without any product the rest alone takes 0.82 of
// the time.  One prompt of 8192 tokens, 32 heads, bf16: 442 us (1245 TFLOP/s),
// 503 to 514 us back to back at the board's power limit; 16 prompts of 1 to 300
// tokens: 17 us.  Two warps per 32 rows, each with half of the columns, are
// slower (485 us: the halves have to meet for every maximum).
// Tensor memory: S0 | S1 | O0 | O1, 128 columns each.  In-order execution of
// the MMAs makes "S_i(j + 1) is complete" mean that O_i is at rest too.
#include <algorithm>
#include <type_traits>

#include "../../include/innerq_b200.h"
#include "common.cuh"
#include "innerq_internal.h"
#include "tcgen05_ptx.cuh"

namespace innerq {
namespace {

constexpr int kRows = 128;               // rows of a query tile, keys of a key tile
constexpr int kHalfTile = kRows * 128;   // bytes of 64 channels of a tile
constexpr int kTileBytes = 2 * kHalfTile;
constexpr int kRing = 5;                 // K and V tiles in flight
constexpr int kThreads = 384;
constexpr float kShift = 7.f;            // P carries 2^7
constexpr float kSlack = 8.f;            // lag of the running maximum
constexpr float kNoMax = -1e30f;
constexpr uint32_t kWait = 1u << 14;
// P is handed over in two parts, so that P V starts before P is complete; the
// first has this many of its four quarters: 508 us with 1, 501 with 2, 497 with
// 3, some 515 in one part (8192 tokens, sustained)
constexpr int kParts = 2, kFirstPart = 3;
// one pair of exponentials of this many goes to the FMA pipe: 472 us of 477
// without (8192 tokens, an earlier state of the kernel), 2.25 ms of 2.38
// (chunks over 8111 tokens); every second pair is slower again (497 us)
constexpr int kPolyOf = 4;

struct PromptDev {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;
  const int32_t* cu_q;
  const int32_t* cu_k;
  uint16_t* out;
  float* lse;
  float scale_log2;  // > 0; `negate` holds the sign
  int negate;
  int B, Hq, Hkv, Tq, Tk, causal, slots;
  int pack, tokens, groups;  // query heads of a row's token, tokens of a tile, groups of heads
};

// One piece of work: two query tiles of one sequence and group of heads, and how
// many key tiles each needs (n0 < 0: there is no more work).
struct Work {
  int head, q_base, nq, k_base, nk, q0, n0, n1;
  int cut;    // from this key tile on, some row must not see all of a tile
  int dirty;  // the scan found values that are not finite
  // keys that query row i of the sequence may see
  __device__ __forceinline__ int limit(int i, int causal) const { return causal ? min(nk, i + nk - nq + 1) : nk; }
};
constexpr int kWorks = 4;  // pieces of work that the CTA's warps may be apart

struct alignas(1024) Smem {
  uint8_t q[2][kTileBytes];
  uint8_t ring[kRing][kTileBytes];
  Work work[kWorks];
  uint4 answer;
  uint64_t work_full[kWorks], work_empty[kWorks], asked;
  uint64_t q_full, q_empty, full[kRing], checked[kRing], empty[kRing], s_full[2], p_ready[2][kParts], o_full[2], drained;
  uint32_t tmem;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// two fp32 values at a time
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2_ftz(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.ftz.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// the larger of three; NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^y of two values (finite, or -inf) on the FMA pipe, which the
// special-function unit's 2^x leaves idle: y = n + f with n the nearest
// integer, a polynomial of degree 4 for 2^f on [-1/2, 1/2] (minimax of the
// relative error, 2.6e-6, from the Remez exchange), and n added to the exponent.
// Values below -127 + 2^-16 count as that: the exponent field is 0 there and the
// result, some 80 units of the smallest subnormal, is 0 in either type and in a
// sum that takes subnormals for 0 (add2_ftz), so -inf has no weight.
__device__ __forceinline__ void exp2_poly(uint64_t y, float& a, float& b) {
  float y0, y1;
  f2_split(y, y0, y1);
  const float least = -127.f + 1.f / 65536.f;
  y = f2(fmaxf(y0, least), fmaxf(y1, least));
  const float big = 12582912.f;  // 1.5 2^23: a sum with it is rounded to an integer
  const uint64_t t = add2(y, f2(big, big)), n = add2(t, f2(-big, -big));
  const uint64_t f = fma2(n, f2(-1.f, -1.f), y);
  uint64_t p = fma2(f, f2(0.009570102207362652f, 0.009570102207362652f), f2(0.05591785907745361f, 0.05591785907745361f));
  p = fma2(p, f, f2(0.240247443318367f, 0.240247443318367f));
  p = fma2(p, f, f2(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(p, f, f2(0.9999992847442627f, 0.9999992847442627f));
  float t0, t1, p0, p1;
  f2_split(t, t0, t1);
  f2_split(p, p0, p1);
  a = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
  b = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}

// two probabilities as one word of the type
template <int DT> __device__ __forceinline__ uint32_t pack_p(float a, float b) {
  uint32_t r;
  if constexpr (DT == F16)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(b), "f"(a));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

// The work of block `block` (the last queries of a sequence see the most keys:
// heavy blocks first); one warp.  False: none, the grid is an upper bound.
__device__ __forceinline__ bool decode(const PromptDev& a, int block, int lane, Work& w) {
  const int slot = a.slots - 1 - block / a.groups, pair = 2 * a.tokens;
  w.head = block % a.groups * a.pack;
  // slots of sequence b start at cu_q[b] / pair + b: room for its pairs of tiles
  int b = -1, lo = 0, hi = 0, k_lo = 0, k_hi = 0;
  for (int i = lane; i < a.B; i += 32) {
    const int x = a.cu_q[i], y = a.cu_q[i + 1], kx = a.cu_k[i], ky = a.cu_k[i + 1];
    if (x >= 0 && x / pair + i <= slot && slot < x / pair + i + (y - x + pair - 1) / pair) b = i, lo = x, hi = y, k_lo = kx, k_hi = ky;
  }
  const uint32_t who = __ballot_sync(~0u, b >= 0);
  if (!who) return false;
  const int src = __ffs(who) - 1;
  b = __shfl_sync(~0u, b, src);
  w.q_base = __shfl_sync(~0u, lo, src);
  w.nq = min(__shfl_sync(~0u, hi, src), a.Tq) - w.q_base;
  w.k_base = max(0, __shfl_sync(~0u, k_lo, src));
  w.nk = max(0, min(__shfl_sync(~0u, k_hi, src), a.Tk) - w.k_base);
  w.q0 = (slot - (w.q_base / pair + b)) * pair;
  if (w.q0 >= w.nq) return false;
  int n[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int first = w.q0 + i * a.tokens, last = min(first + a.tokens, w.nq) - 1;
    n[i] = ((first < w.nq ? max(0, w.limit(last, a.causal)) : 0) + kRows - 1) / kRows;
  }
  w.n0 = n[0];
  w.n1 = n[1];
  w.cut = max(0, w.limit(w.q0 + (n[0] > 0 ? 0 : a.tokens), a.causal)) / kRows;
  w.dirty = 0;
  return true;
}

// A warp's way through the CTA's pieces of work.
struct Pieces {
  Smem& sm;
  int slot = 0;
  uint32_t parity = 0;
  bool ok = true;
  __device__ __forceinline__ Pieces(Smem& s) : sm(s) {}
  // the next piece; null: no more (or, with ok false, a wait that ran out)
  __device__ __forceinline__ Work* next() {
    ok = mbar_wait_warp(&sm.work_full[slot], parity, kWait);
    Work* w = &sm.work[slot];
    return ok && w->n0 >= 0 ? w : nullptr;
  }
  __device__ __forceinline__ void step() {
    if (++slot == kWorks) slot = 0, parity ^= 1;
  }
  __device__ __forceinline__ void done(int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.work_empty[slot]);
    step();
  }
};

// Four lanes swap 16-byte pieces w[0..3] so that lane k ends with piece k of
// the rows of all four: a 4 x 4 transpose in two exchanges.
__device__ __forceinline__ void transpose4(uint4 w[4], int lane) {
#pragma unroll
  for (int bit = 1; bit <= 2; bit <<= 1) {
    const bool up = lane & bit;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t* lo = reinterpret_cast<uint32_t*>(&w[bit == 1 ? 2 * x : x]);
      uint32_t* hi = reinterpret_cast<uint32_t*>(&w[bit == 1 ? 2 * x + 1 : x + 2]);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t got = __shfl_xor_sync(~0u, up ? lo[y] : hi[y], bit);
        if (up)
          lo[y] = got;
        else
          hi[y] = got;
      }
    }
  }
}

// The finished rows of a warp, one per thread: O / l, or zeros where there is
// no O.  Four lanes write 64 contiguous bytes of a row (a thread on its own
// would spread every store over 32 rows: 2.5 us per piece of work).  True: this
// thread's row holds something that is not finite (fp16; not looked for in bf16).
template <int DT>
__device__ __forceinline__ bool write_rows(uint32_t to, bool any, float inv, uint16_t* out, int lane) {
  __half2 seen = __half2half2(__half(0.f));
  uint64_t row[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) row[x] = __shfl_sync(~0u, (unsigned long long)out, (lane & ~3) + x);
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    float o[32];
    if (any) {
      tmem_ld32(to + 32 * c, o);
      tmem_wait_ld();
    } else {
#pragma unroll
      for (int x = 0; x < 32; ++x) o[x] = 0.f;
    }
    uint4 w[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      uint32_t* e = reinterpret_cast<uint32_t*>(&w[x]);
#pragma unroll
      for (int y = 0; y < 4; ++y) e[y] = inv == 0.f ? 0u : pack_p<DT>(o[8 * x + 2 * y] * inv, o[8 * x + 2 * y + 1] * inv);
      if constexpr (DT == F16) {
#pragma unroll
        for (int y = 0; y < 4; ++y) seen = __hfma2(as_pair<F16>(e[y]), __half2half2(__half(0.f)), seen);
      }
    }
    transpose4(w, lane);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (row[x]) reinterpret_cast<uint4*>(row[x])[4 * c + (lane & 3)] = w[x];
  }
  return DT == F16 && !__hbeq2(seen, seen);
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv, PromptDev a) {
  extern __shared__ __align__(1024) uint8_t raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31;  // warp: uniform, and known to be

  if (tid == 0) {
    for (int i = 0; i < kWorks; ++i) {
      mbar_init(&sm.work_full[i], 1);
      mbar_init(&sm.work_empty[i], 11);
    }
    mbar_init(&sm.asked, 1);
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    mbar_init(&sm.drained, 1);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.checked[i], 2);
      mbar_init(&sm.empty[i], 3);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.s_full[i], 1);
      for (int x = 0; x < kParts; ++x) mbar_init(&sm.p_ready[i][x], 4);
      mbar_init(&sm.o_full[i], 1);
    }
    mbar_fence_init();
  }
  if (tid == 9 * 32) {
    tma_prefetch(&mq);
    tma_prefetch(&mk);
    tma_prefetch(&mv);
  }
  if (warp == 8) tmem_alloc(&sm.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  griddep_wait();
  griddep_launch_dependents();

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
    Pieces pieces(sm);
    if (warp == 9) {
      // -------------------------------------------------------- TMA loads
      int st = 0, filled = 0, q_count = 0;  // ring slot of the next tile, how many are in use at most
      uint32_t parity = 1;                  // of the slot's last release
      bool ok = true;
      while (Work* w = pieces.next()) {
        const int n = max(w->n0, w->n1), tiles = w->n1 > 0 ? 2 : 1, head = w->head, q_row = w->q_base + w->q0, k_base = w->k_base;
        pieces.done(lane);
        if (n == 0) continue;
        const int kv_head = head / (a.Hq / a.Hkv);
        if (q_count > 0) ok = mbar_wait_warp(&sm.q_empty, (q_count - 1) & 1, kWait);
        if (!ok) break;
        ++q_count;
        if (lane == 0) {
          mbar_arrive_tx(&sm.q_full, tiles * a.tokens * a.pack * 256);
          for (int i = 0; i < tiles; ++i)
            for (int h = 0; h < 2; ++h) tma_load_3d(sm.q[i] + h * kHalfTile, &mq, 64 * h, head, q_row + i * a.tokens, &sm.q_full);
        }
        for (int it = 0; ok && it < 2 * n; ++it) {
          if (filled == kRing)
            ok = mbar_wait_warp(&sm.empty[st], parity, kWait);
          else
            ++filled;
          if (ok && lane == 0) {
            const CUtensorMap* m = it & 1 ? &mv : &mk;
            mbar_arrive_tx(&sm.full[st], kTileBytes);
            for (int h = 0; h < 2; ++h)
              tma_load_3d(sm.ring[st] + h * kHalfTile, m, 64 * h, kv_head, k_base + (it >> 1) * kRows, &sm.full[st]);
          }
          if (++st == kRing) st = 0, parity ^= 1;
        }
        if (!ok) break;
      }
      if (!ok || !pieces.ok) {
        // give up: the copies under way must land before the memory is given
        // away.  `parity` is that of the releases; the fillings before slot st
        // have the same one, those from st on the other.
        if (q_count > 0) mbar_wait_bounded(&sm.q_full, (q_count - 1) & 1, kWait / 16);
        for (int i = 0; i < filled; ++i) mbar_wait_bounded(&sm.full[i], i < st ? parity ^ 1 : parity, kWait / 16);
      }
    } else if (warp == 8) {
      // -------------------------------------------------------------- MMAs
      constexpr uint32_t id_s = mma_idesc(kRows, kRows, DT, 0), id_o = mma_idesc(kRows, 128, DT, 1), hi = desc_hi(1024);
      const uint32_t leader = elect_one();
      const uint32_t tm = __shfl_sync(~0u, tmem, 0), q_lo = __shfl_sync(~0u, desc_lo(smem_u32(sm.q[0]), 16), 0),
                     k_lo = __shfl_sync(~0u, desc_lo(smem_u32(sm.ring[0]), 16), 0),
                     v_lo = __shfl_sync(~0u, desc_lo(smem_u32(sm.ring[0]), kHalfTile), 0);
      auto scores = [&](int i, int st) {
        const uint32_t da = q_lo + i * (kTileBytes >> 4), db = k_lo + st * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t step = (k & 3) * 2 + (k >> 2) * (kHalfTile >> 4);
          mma_ss<hi, hi>(leader, tm + i * 128, da + step, db + step, id_s, k > 0);
        }
        mma_commit(leader, &sm.s_full[i]);
      };
      auto values = [&](int i, int st, int part, uint32_t acc) {
        const uint32_t db = v_lo + st * (kTileBytes >> 4);
#pragma unroll
        for (int k = part ? 2 * kFirstPart : 0; k < (part ? 8 : 2 * kFirstPart); ++k)
          mma_ts<hi>(leader, tm + 256 + i * 128, tm + i * 128 + 8 * k, db + k * (2048 >> 4), id_o, k > 0 ? 1u : acc);
      };
      // ring slots of K_j / V_j in turn, with the parities of their fillings
      int st = 0;
      uint32_t par = 0, q_par = 0, p_par[2] = {0, 0};
      auto advance = [&]() {
        if (++st == kRing) st = 0, par ^= 1;
      };
      bool ok = true;
      while (Work* w = pieces.next()) {
        const int n0 = __shfl_sync(~0u, w->n0, 0), n1 = __shfl_sync(~0u, w->n1, 0), cut = __shfl_sync(~0u, w->cut, 0);
        const int n = max(n0, n1);
        pieces.done(lane);
        if (n == 0) continue;
        ok = mbar_wait_bounded(&sm.q_full, q_par, kWait) && mbar_wait_bounded(&sm.full[st], par, kWait);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        q_par ^= 1;
        tc_fence_after();
        if (n0 > 0) scores(0, st);
        if (n1 > 0) scores(1, st);
        mma_commit(leader, &sm.empty[st]);
        if (n == 1) mma_commit(leader, &sm.q_empty);
        advance();
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
          const int vs = st;
          const uint32_t vp = par;
          advance();
          const int ks = st;
          const uint32_t kp = par;
          ok = mbar_wait_bounded(&sm.full[vs], vp, kWait);
          if (j >= cut) ok = ok && mbar_wait_bounded(&sm.checked[vs], vp, kWait);
          const uint32_t acc = j > 0;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int ni = i ? n1 : n0;
            if (j < ni) {
#pragma unroll
              for (int x = 0; x < kParts; ++x) {
                ok = ok && mbar_wait_bounded(&sm.p_ready[i][x], p_par[i], kWait);
                if (x == kParts - 1 && j + 1 < ni) ok = ok && mbar_wait_bounded(&sm.full[ks], kp, kWait);
                ok = __all_sync(~0u, ok);
                if (ok) {
                  tc_fence_after();
                  values(i, vs, x, acc);
                }
              }
              p_par[i] ^= 1;
              if (ok) {
                if (j + 1 < ni)
                  scores(i, ks);
                else
                  mma_commit(leader, &sm.o_full[i]);
              }
            }
          }
          if (!ok) break;
          mma_commit(leader, &sm.empty[vs]);
          if (j + 1 < n) {
            mma_commit(leader, &sm.empty[ks]);
            if (j + 2 == n) mma_commit(leader, &sm.q_empty);  // the last scores are under way
            advance();
          }
        }
        if (!ok) break;
      }
      // no arrival may be outstanding when the CTA ends
      mma_commit(leader, &sm.drained);
      mbar_wait_bounded(&sm.drained, 0, kWait);
    } else {
      // ------------------ warps 10, 11: values that are not finite; 11: more work
      bool asking = true;
      uint32_t asked_par = 0;
      int put = 0;
      uint32_t put_par = 1;
      // publish the next piece of work; the first is this block's own
      auto publish = [&](int block) {
        Work w;
        bool any = block >= 0 && decode(a, block, lane, w);
        while (!any && asking) {
          if (lane == 0) {
            mbar_arrive_tx(&sm.asked, 16);
            next_block_ask(&sm.answer, &sm.asked);
          }
          __syncwarp();
          asking = mbar_wait_warp(&sm.asked, asked_par, kWait);
          asked_par ^= 1;
          const int x = asking ? next_block_get(&sm.answer) : -1;
          fence_proxy_async();
          __syncwarp();
          asking = x >= 0;
          any = asking && decode(a, x, lane, w);
        }
        if (!any) w.n0 = -1;
        if (!mbar_wait_warp(&sm.work_empty[put], put_par, kWait)) return;
        if (lane == 0) {
          sm.work[put] = w;
          mbar_arrive(&sm.work_full[put]);
        }
        __syncwarp();
        if (++put == kWorks) put = 0, put_par ^= 1;
      };
      if (warp == 11) publish(blockIdx.x);
      int st = 0;
      uint32_t par = 0;
      bool ok = true;
      while (Work* w = pieces.next()) {
        const int n = max(w->n0, w->n1), cut = w->cut;
        if (warp == 11) publish(-1);
        for (int it = 0; ok && it < 2 * n; ++it) {
          ok = mbar_wait_warp(&sm.full[st], par, kWait);
          if (!ok) break;
          if ((it & 1) && (it >> 1) >= cut) {
            uint4* p = reinterpret_cast<uint4*>(sm.ring[st]) + (warp - 10) * (kTileBytes / 32);
            bool found = false;
#pragma unroll 4
            for (int x = lane; x < kTileBytes / 32; x += 32) {
              uint4 v = p[x];
              uint32_t* e = reinterpret_cast<uint32_t*>(&v);
              bool bad = false;
#pragma unroll
              for (int y = 0; y < 4; ++y) bad |= not_finite<DT>(e[y]) | not_finite<DT>(e[y] >> 16);
              if (bad) {
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  e[y] &= (not_finite<DT>(e[y]) ? 0u : 0xffffu) | (not_finite<DT>(e[y] >> 16) ? 0u : 0xffff0000u);
                p[x] = v;
                found = true;
              }
            }
            if (found) {
              w->dirty = 1;
              fence_proxy_async();
            }
          }
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&sm.checked[st]);
            mbar_arrive(&sm.empty[st]);
          }
          if (++st == kRing) st = 0, par ^= 1;
        }
        if (!ok) break;
        if (warp == 10)
          pieces.done(lane);
        else
          pieces.step();
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;\n");
    // ------------------------------------------------------------- softmax
    const int i = warp >> 2, row = tid & 127, tok = row / a.pack, sub = row % a.pack;  // row: token, then head
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // 32 lanes per warp
    const uint32_t ts = tmem + i * 128 + lanes, to = tmem + 256 + i * 128 + lanes;
    const uint64_t scale = f2(a.scale_log2, a.scale_log2);
    Pieces pieces(sm);
    uint32_t s_par = 0, o_par = 0;
    while (Work* w = pieces.next()) {
      const int first = w->q0 + i * a.tokens, n = i ? w->n1 : w->n0, qi = first + tok;
      const bool real = tok < a.tokens && qi < w->nq;
      const int lim = real ? w->limit(qi, a.causal) : 0x7fffffff, head = w->head + sub;
      float m = kNoMax, l = 0.f;
      bool ok = true;
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        ok = mbar_wait_warp(&sm.s_full[i], s_par, kWait);
        if (!ok) break;
        s_par ^= 1;
        tc_fence_after();
        float s[128];
        const int seen = lim - kRows * j;
        const bool whole = __all_sync(~0u, seen >= kRows);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, s + 32 * c);
        tmem_wait_ld();
        if (a.negate) {
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = -s[c];
        }
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = c < seen ? s[c] : -INFINITY;
        }
        float t4[4];
#pragma unroll
        for (int c = 0; c < 128; c += 8) {
#pragma unroll
          for (int x = 0; x < 4; ++x) t4[x] = max3(c ? t4[x] : s[2 * x], s[c + 2 * x], s[c + 2 * x + 1]);
        }
        // a row without a query (another sequence's, or bits that nothing wrote)
        // has no say in what the warp does with the others
        const float t = real ? max3(max3(t4[0], t4[1], t4[2]), t4[3], t4[3]) * a.scale_log2 : -INFINITY;
        // no logit is NaN or +inf: some exponentials may take the FMA pipe
        const bool mixed = !whole ? false : __all_sync(~0u, t < INFINITY);
        if (__any_sync(~0u, t > m + kSlack)) {
          const float mn = fmaxf(m, t), corr = ex2(m - mn);
          m = mn;
          l *= corr;
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              float o[32];
              tmem_ld32(to + 32 * c, o);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] *= corr;
              tmem_st32(to + 32 * c, o);
            }
          }
        }
        const uint64_t base = f2(kShift - m, kShift - m);
        uint64_t sum[2] = {0, 0};
        auto probabilities = [&](auto poly) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const uint64_t y = fma2(f2(s[32 * c + 2 * x], s[32 * c + 2 * x + 1]), scale, base);
              float p0, p1;
              if (decltype(poly)::value && x % kPolyOf == kPolyOf - 1) {
                exp2_poly(y, p0, p1);
              } else {
                f2_split(y, p0, p1);
                p0 = ex2(p0);
                p1 = ex2(p1);
              }
              sum[x & 1] = add2_ftz(sum[x & 1], f2(p0, p1));
              p[x] = pack_p<DT>(p0, p1);
            }
            tmem_st16(ts + 16 * c, p);
            if (c == kFirstPart - 1 || c == 3) {
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&sm.p_ready[i][c == 3]);
            }
          }
        };
        if (mixed)
          probabilities(std::true_type{});
        else
          probabilities(std::false_type{});
        float l0, l1;
        f2_split(add2(sum[0], sum[1]), l0, l1);
        l += l0 + l1;
      }
      // ---------------------------------------------------------- epilogue
      if (first < w->nq) {
        if (n > 0) {
          if (ok) ok = mbar_wait_warp(&sm.o_full[i], o_par, kWait);
          o_par ^= 1;
          tc_fence_after();
        }
        // a row that sees no key is 0; one that does, but whose logits are all
        // -inf, is 0 / 0
        const float inv = !ok ? NAN : lim <= 0 ? 0.f : l != 0.f ? 1.f / l : NAN;
        uint16_t* out = a.out + (int64_t)(w->q_base + qi) * a.o_st + head * a.o_sh;
        const bool odd = write_rows<DT>(to, n > 0, inv, real ? out : nullptr, lane);
        tc_fence_before();
        __syncwarp();
        // Values that are not finite, one by one (the row was written by this
        // warp's lanes: made visible by the warp barrier).
        const bool dirty = *(volatile int*)&w->dirty, fine = ok && real && inv == inv;
        const int keys = fine ? min(kRows * n, lim) : 0;
        if (__any_sync(~0u, fine && (dirty || (DT == F16 && odd)))) {
          const int kv_head = w->head / (a.Hq / a.Hkv);
          const uint16_t* qr = a.q + (int64_t)(w->q_base + qi) * a.q_st + head * a.q_sh;
          auto value_row = [&](int key) { return a.v + (int64_t)(w->k_base + key) * a.v_st + kv_head * a.v_sh; };
          auto weight = [&](int key) {
            const uint16_t* kr = a.k + (int64_t)(w->k_base + key) * a.k_st + kv_head * a.k_sh;
            float dot = 0.f;
            for (int x = 0; x < kD; ++x) dot = fmaf(to_f<DT>(qr[x]), to_f<DT>(kr[x]), dot);
            return ex2(fmaf(a.negate ? -dot : dot, a.scale_log2, kShift - m)) * inv;
          };
          if (DT == F16 && __any_sync(~0u, fine && odd)) {
            // An infinity times a probability that is 0 in fp16, but not 0, left
            // NaN.  Such channels (lost) start again from 0 and take all values
            // that are not finite until they are NaN for good; the lanes look for
            // keys with such values, 32 at a time.
            uint32_t lost[kD / 32];
#pragma unroll
            for (int x = 0; x < kD / 32; ++x) {
              lost[x] = 0;
              for (int y = 0; fine && odd && y < 32; ++y)
                if (to_f<DT>(out[32 * x + y]) != to_f<DT>(out[32 * x + y])) {
                  lost[x] |= 1u << y;
                  out[32 * x + y] = 0;
                }
            }
            const int most = __reduce_max_sync(~0u, keys);
            for (int key0 = 0; key0 < most && __any_sync(~0u, lost[0] | lost[1] | lost[2] | lost[3]); key0 += 32) {
              bool found = false;
              if (key0 + lane < most) {
                const uint4* row4 = reinterpret_cast<const uint4*>(value_row(key0 + lane));
                for (int x = 0; x < kD / 8; ++x) {
                  const uint4 v = row4[x];
                  const uint32_t* e = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
                  for (int y = 0; y < 4; ++y) found |= not_finite<DT>(e[y]) | not_finite<DT>(e[y] >> 16);
                }
              }
              for (uint32_t hits = __ballot_sync(~0u, found); hits; hits &= hits - 1) {
                const int key = key0 + __ffs(hits) - 1;
                if (key >= keys || !(lost[0] | lost[1] | lost[2] | lost[3])) continue;
                const uint16_t* vr = value_row(key);
                float p = -1.f;
#pragma unroll
                for (int x = 0; x < kD / 32; ++x)
                  for (uint32_t left = lost[x]; left; left &= left - 1) {
                    const int d = 32 * x + __ffs(left) - 1;
                    const float v = to_f<DT>(vr[d]);
                    // (once more the same infinity: a sum of 100000 keys would
                    // take their weights otherwise)
                    if (!not_finite<DT>(vr[d]) || v == to_f<DT>(out[d])) continue;
                    if (p == -1.f) p = weight(key);
                    const float sum = fmaf(p, v, to_f<DT>(out[d]));
                    out[d] = from_f<DT>(sum);
                    if (sum != sum) lost[x] &= ~(left & (0u - left));
                  }
              }
              __syncwarp();
            }
          }
          // values that were set to 0 and that this row does see
          for (int key = kRows * w->cut; dirty && key < keys; ++key) {
            const uint16_t* vr = value_row(key);
            float p = -1.f;
            for (int d = 0; d < kD; ++d) {
              if (!not_finite<DT>(vr[d])) continue;
              if (p == -1.f) p = weight(key);
              out[d] = from_f<DT>(to_f<DT>(out[d]) + p * to_f<DT>(vr[d]));
            }
          }
        }
        if (a.lse && real)
          a.lse[(int64_t)(w->q_base + qi) * a.Hq + head] = l == 0.f || lim <= 0 ? -INFINITY : m - kShift + log2f(l);
      }
      if (!ok) break;
      pieces.done(lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_free(tmem, 512);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeFn)p;
  }();
  return fn;
}

// boxes of `tokens` tokens x `heads` heads x 64 channels of [T][H][128]
bool encode(CUtensorMap* m, const void* base, int dtype, int H, int T, int64_t sh, int64_t st, int heads, int tokens) {
  const EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)kD, (cuuint64_t)H, (cuuint64_t)T};
  // a dimension of one element has no stride of its own
  const cuuint64_t strides[2] = {(cuuint64_t)(H > 1 ? sh : kD) * 2, (cuuint64_t)(T > 1 ? st : kD) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens}, one[3] = {1, 1, 1};
  return fn(m, dtype == INNERQ_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT>
cudaError_t launch_prompt(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PromptDev& a,
                          cudaStream_t s) {
  static bool ready[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  constexpr int smem = sizeof(Smem) + 1024;
  if (dev >= 64 || !ready[dev]) {
    e = cudaFuncSetAttribute(prompt_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready[dev] = true;
  }
  return launch_pdl(prompt_kernel<DT>, dim3((unsigned)a.slots * a.groups), dim3(kThreads), smem, s, mq, mk, mv, a);
}

}  // namespace
}  // namespace innerq

using namespace innerq;

extern "C" int innerq_prompt_attn(const innerq_prompt_args* p, void* stream) {
  if (!p) return set_last_error(INNERQ_ERR_ARG, "null args");
  if (p->struct_size != (int32_t)sizeof(innerq_prompt_args))
    return set_last_error(INNERQ_ERR_ARG, "struct_size %d != %d (ABI mismatch)", p->struct_size, (int)sizeof(innerq_prompt_args));
  if (p->dtype != INNERQ_DT_F16 && p->dtype != INNERQ_DT_BF16) return set_last_error(INNERQ_ERR_ARG, "dtype %d", p->dtype);
  if (p->D != kD) return set_last_error(INNERQ_ERR_UNSUPPORTED, "head_dim %d (only 128 is built)", p->D);
  if (p->B < 0 || p->Tq < 0 || p->Tk < 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Hq % p->Hkv)
    return set_last_error(INNERQ_ERR_ARG, "sizes: %d sequences, %d queries, %d keys, %d / %d heads", p->B, p->Tq, p->Tk, p->Hq, p->Hkv);
  if (p->B == 0 || p->Tq == 0) return INNERQ_OK;
  if (!p->q || !p->out || !p->cu_q || !p->cu_k || (p->Tk > 0 && (!p->k || !p->v)))
    return set_last_error(INNERQ_ERR_ARG, "null pointer");
  const int64_t st[] = {p->q_st, p->q_sh, p->k_st, p->k_sh, p->v_st, p->v_sh, p->o_st, p->o_sh};
  for (int64_t x : st)
    if (x % 8 || x < 0) return set_last_error(INNERQ_ERR_ARG, "strides must be multiples of 8 elements");
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->out))
    return set_last_error(INNERQ_ERR_ARG, "rows must be 16-byte aligned");
  PromptDev a;
  a.q = (const uint16_t*)p->q; a.k = (const uint16_t*)p->k; a.v = (const uint16_t*)p->v;
  a.q_st = p->q_st; a.q_sh = p->q_sh; a.k_st = p->k_st; a.k_sh = p->k_sh;
  a.v_st = p->v_st; a.v_sh = p->v_sh; a.o_st = p->o_st; a.o_sh = p->o_sh;
  a.cu_q = p->cu_q; a.cu_k = p->cu_k;
  a.out = (uint16_t*)p->out;
  a.lse = p->lse;
  // a scale of 0 weighs all keys alike; masked logits are -inf, and -inf * 0 is NaN
  a.scale_log2 = (p->scale < 0 ? -p->scale : p->scale) * 1.4426950408889634f;
  if (a.scale_log2 < 1e-37f) a.scale_log2 = 1e-37f;  // (NaN stays)
  a.negate = p->scale < 0;
  a.B = p->B; a.Hq = p->Hq; a.Hkv = p->Hkv; a.Tq = p->Tq; a.Tk = p->Tk; a.causal = p->causal;
  // The rows of a query tile are tokens times the query heads that share their
  // keys, so short prompts fill tiles too.
  const int ratio = p->Hq / p->Hkv;
  a.pack = ratio <= 32 ? ratio : 1;
  a.tokens = kRows / a.pack;
  a.groups = p->Hq / a.pack;
  a.slots = p->Tq / (2 * a.tokens) + p->B;
  if ((int64_t)a.slots * a.groups > 0x7fffffff) return set_last_error(INNERQ_ERR_ARG, "too many blocks for one launch");
  CUtensorMap mq, mk, mv;
  const bool none = p->Tk == 0;  // no keys: the maps are never used
  if (!encode(&mq, p->q, p->dtype, p->Hq, p->Tq, p->q_sh, p->q_st, a.pack, a.tokens) ||
      !encode(&mk, none ? p->q : p->k, p->dtype, none ? 1 : p->Hkv, none ? 1 : p->Tk, p->k_sh, p->k_st, 1, kRows) ||
      !encode(&mv, none ? p->q : p->v, p->dtype, none ? 1 : p->Hkv, none ? 1 : p->Tk, p->v_sh, p->v_st, 1, kRows))
    return set_last_error(INNERQ_ERR_ARG, "q, k and v: strides or sizes that a tensor map cannot describe");
  const cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = p->dtype == INNERQ_DT_BF16 ? launch_prompt<BF16>(mq, mk, mv, a, s) : launch_prompt<F16>(mq, mk, mv, a, s);
  return e == cudaSuccess ? INNERQ_OK : set_last_error(INNERQ_ERR_CUDA, "prompt_attn: %s", cudaGetErrorString(e));
}
