// Attention of whole prompts packed one behind the other.
#include "../../include/innerq_b200.h"
#include "common.cuh"
#include "innerq_internal.h"

namespace innerq {
namespace {

struct PromptDev {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;
  const int32_t* cu_q;
  const int32_t* cu_k;
  uint16_t* out;
  float* lse;
  float scale_log2;
  int B, Hq, Hkv, Tq, Tk, causal;
};

// One warp per (query, head), four channels per lane.
template <int DT>
__global__ void __launch_bounds__(128) prompt_simple_kernel(PromptDev a) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, h = blockIdx.y, t = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= a.Tq) return;
  int b = -1;
  for (int i = 0; i < a.B; ++i)
    if (a.cu_q[i] <= t && t < a.cu_q[i + 1]) b = i;
  if (b < 0) return;
  const int k0 = max(0, a.cu_k[b]), nk = min(a.cu_k[b + 1], a.Tk) - k0;
  const int seen = a.causal ? min(nk, t - a.cu_q[b] + 1 + nk - (a.cu_q[b + 1] - a.cu_q[b])) : nk;
  float qf[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) qf[i] = to_f<DT>(a.q[t * a.q_st + h * a.q_sh + 4 * lane + i]);
  const int hk = h / (a.Hq / a.Hkv);
  for (int j = 0; j < seen; ++j) {
    const uint2 kw = *reinterpret_cast<const uint2*>(a.k + (k0 + j) * a.k_st + hk * a.k_sh + 4 * lane);
    const uint2 vw = *reinterpret_cast<const uint2*>(a.v + (k0 + j) * a.v_st + hk * a.v_sh + 4 * lane);
    float s = qf[0] * to_f<DT>(kw.x & 0xffff) + qf[1] * to_f<DT>(kw.x >> 16) + qf[2] * to_f<DT>(kw.y & 0xffff) +
              qf[3] * to_f<DT>(kw.y >> 16);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    s *= a.scale_log2;
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn, corr = exp2f(m - base), p = exp2f(s - base);
    l = l * corr + p;
    acc[0] = acc[0] * corr + p * to_f<DT>(vw.x & 0xffff);
    acc[1] = acc[1] * corr + p * to_f<DT>(vw.x >> 16);
    acc[2] = acc[2] * corr + p * to_f<DT>(vw.y & 0xffff);
    acc[3] = acc[3] * corr + p * to_f<DT>(vw.y >> 16);
    m = mn;
  }
  const float inv = seen > 0 ? 1.f / l : 0.f;
  uint2 o;
  o.x = pack2(from_f<DT>(acc[0] * inv), from_f<DT>(acc[1] * inv));
  o.y = pack2(from_f<DT>(acc[2] * inv), from_f<DT>(acc[3] * inv));
  *reinterpret_cast<uint2*>(a.out + t * a.o_st + h * a.o_sh + 4 * lane) = o;
  if (a.lse && lane == 0) a.lse[(int64_t)t * a.Hq + h] = m + log2f(l);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

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
    if (x % 8) return set_last_error(INNERQ_ERR_ARG, "strides must be multiples of 8 elements");
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->out))
    return set_last_error(INNERQ_ERR_ARG, "rows must be 16-byte aligned");
  if (p->Hq > 65535) return set_last_error(INNERQ_ERR_ARG, "more than 65535 heads");
  PromptDev a{(const uint16_t*)p->q, (const uint16_t*)p->k, (const uint16_t*)p->v, p->q_st, p->q_sh, p->k_st, p->k_sh,
              p->v_st, p->v_sh, p->o_st, p->o_sh, p->cu_q, p->cu_k, (uint16_t*)p->out, p->lse,
              p->scale * 1.4426950408889634f, p->B, p->Hq, p->Hkv, p->Tq, p->Tk, p->causal};
  const dim3 grid((p->Tq + 3) / 4, p->Hq);
  const cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = p->dtype == INNERQ_DT_BF16 ? launch_pdl(prompt_simple_kernel<BF16>, grid, dim3(128), 0, s, a)
                                                   : launch_pdl(prompt_simple_kernel<F16>, grid, dim3(128), 0, s, a);
  return e == cudaSuccess ? INNERQ_OK : set_last_error(INNERQ_ERR_CUDA, "prompt_attn: %s", cudaGetErrorString(e));
}
