// Decode attention over the paged 4-bit cache: one query token per sequence,
// a length per sequence.
#include "innerq_internal.h"
#include "paged.cuh"

namespace innerq {
namespace {

struct AttnDev {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  uint16_t* out;
  int64_t o_sb, o_sh;
  float* lse;
  float scale_log2;
  int Hq, R;
};

// One block per (sequence, KV head): a tile of 32 tokens at a time is expanded
// to fp32 in shared memory; online softmax over the tiles.
template <int DT>
__global__ void __launch_bounds__(128) attn_simple_kernel(PagedDev c, AttnDev a) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ float kt[32][kD + 1], vt[32][kD], p[8][32], qs[8][kD], corr[8], ms[8], ls[8];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int len = max(0, c.lens[b]), np = c.n_packed(len);
  for (int r = 0; r < a.R; ++r) qs[r][tid] = to_f<DT>(a.q[b * a.q_sb + (h * a.R + r) * a.q_sh + tid]);
  if (tid < 8) ms[tid] = -INFINITY, ls[tid] = 0.f;
  float acc[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) acc[r] = 0.f;
  const int64_t base = c.dense_base(b, h);
  for (int t0 = 0; t0 < len; t0 += 32) {
    __syncthreads();
    const bool packed = t0 >= c.w_sink && t0 - c.w_sink < np;
    const uint8_t* blk = packed ? c.tile(b, h, (t0 - c.w_sink) >> 5) : nullptr;
    const int d = tid;
    for (int r = 0; r < 32; ++r) {
      float kv = NAN, vv = NAN;
      if (packed && blk != nullptr) {
        const uint32_t wk = reinterpret_cast<const uint32_t*>(blk)[(r * 4 + ((d >> 3) & 3)) * 4 + (d >> 5)];
        const float sk = to_f<DT>(reinterpret_cast<const uint16_t*>(blk + kKScale)[(r & 7) * 16 + (r >> 3) * 4 + (d >> 5)]);
        kv = (float)((int)((wk >> (4 * (d & 7))) & 15u) - 8) * sk;
        const int wi = ((((d >> 2) & 3) * 8 + (d >> 4)) * 4 + ((r >> 1) & 3)) * 4 + (d & 3);
        const uint32_t wv = reinterpret_cast<const uint32_t*>(blk + kVCodes)[wi];
        vv = (float)((int)((wv >> (4 * ((r >> 3) + 4 * (r & 1)))) & 15u) - 8) *
             to_f<DT>(reinterpret_cast<const uint16_t*>(blk + kVScale)[d]);
      } else if (!packed && base >= 0) {
        const int64_t at = base + (int64_t)c.row_of(t0 + r) * kD + d;
        kv = to_f<DT>(c.dk[at]);
        vv = to_f<DT>(c.dv[at]);
      }
      kt[r][d] = kv;
      vt[r][d] = t0 + r < len ? vv : 0.f;
    }
    __syncthreads();
    for (int i = tid; i < a.R * 32; i += 128) {
      const int r = i >> 5, t = i & 31;
      float s = 0.f;
      for (int x = 0; x < kD; ++x) s += qs[r][x] * kt[t][x];
      p[r][t] = t0 + t < len ? s * a.scale_log2 : -INFINITY;
    }
    __syncthreads();
    if (tid < a.R) {
      float m = ms[tid];
      for (int t = 0; t < 32; ++t) m = fmaxf(m, p[tid][t]);
      const float base_m = m == -INFINITY ? 0.f : m;
      corr[tid] = exp2f(ms[tid] - base_m);
      float l = ls[tid] * corr[tid];
      for (int t = 0; t < 32; ++t) l += p[tid][t] = exp2f(p[tid][t] - base_m);
      ms[tid] = m;
      ls[tid] = l;
    }
    __syncthreads();
    for (int r = 0; r < a.R; ++r) {
      float s = acc[r] * corr[r];
      for (int t = 0; t < 32; ++t) s += p[r][t] * vt[t][tid];
      acc[r] = s;
    }
  }
  __syncthreads();
  for (int r = 0; r < a.R; ++r) {
    const int hq = h * a.R + r;
    a.out[b * a.o_sb + hq * a.o_sh + tid] = from_f<DT>(len > 0 ? acc[r] / ls[r] : 0.f);
    if (a.lse && tid == 0) a.lse[(int64_t)b * a.Hq + hq] = ms[r] + log2f(ls[r]);
  }
}

}  // namespace
}  // namespace innerq

using namespace innerq;

extern "C" int64_t innerq_paged_attn_workspace(const innerq_paged* cache, int Hq) {
  PagedDev c;
  if (paged_dev(cache, c)) return -1;
  return 256;
}

extern "C" int innerq_paged_attn(const innerq_paged* cache, int Hq, const void* q, int64_t q_sb, int64_t q_sh, float scale,
                                 void* workspace, int64_t workspace_bytes, void* out, int64_t o_sb, int64_t o_sh,
                                 float* lse, void* stream) {
  PagedDev c;
  if (int rc = paged_dev(cache, c)) return rc;
  if (Hq <= 0 || Hq % c.Hkv) return set_last_error(INNERQ_ERR_ARG, "%d query heads over %d key heads", Hq, c.Hkv);
  if (Hq / c.Hkv > 8) return set_last_error(INNERQ_ERR_UNSUPPORTED, "GQA ratio %d (1 to 8 are built)", Hq / c.Hkv);
  if (c.B == 0) return INNERQ_OK;
  if (!q || !out) return set_last_error(INNERQ_ERR_ARG, "null pointer");
  if (((uintptr_t)q & 15) || ((uintptr_t)out & 15) || q_sb % 8 || q_sh % 8 || o_sb % 8 || o_sh % 8)
    return set_last_error(INNERQ_ERR_ARG, "rows must be 16-byte aligned");
  if (c.B > 65535) return set_last_error(INNERQ_ERR_ARG, "more than 65535 sequences");
  AttnDev a{(const uint16_t*)q, q_sb, q_sh, (uint16_t*)out, o_sb, o_sh, lse, scale * 1.4426950408889634f, Hq, Hq / c.Hkv};
  const dim3 grid(c.Hkv, c.B);
  const cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = cache->dtype == INNERQ_DT_BF16 ? launch_pdl(attn_simple_kernel<BF16>, grid, dim3(128), 0, s, c, a)
                                                       : launch_pdl(attn_simple_kernel<F16>, grid, dim3(128), 0, s, c, a);
  return e == cudaSuccess ? INNERQ_OK : set_last_error(INNERQ_ERR_CUDA, "paged_attn: %s", cudaGetErrorString(e));
}
