// fa8_decode.cu — attention of the last few tokens of every sequence over a
// paged e4m3 cache (fa8_decode). No counterpart in the reference.
//
//   s_j = scale * q . k_j,  o = sum_j exp(s_j) v_j / sum_j exp(s_j),
// over the keys j <= position of the query, in one pass with a running
// maximum and sum (fp32). First form: one block per query row, a warp per
// key, lanes over the head dimension.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "fa8_kv.cuh"
#include "sm100_ptx.cuh"

namespace fa8 {
namespace dec {

struct Args {
  kv::CacheView c;
  const char* q;
  char* o;
  float* lse;
  int heads, seqlen_q, prefix_len;
  long long q_sb, q_sh, q_ss, o_sb, o_sh, o_ss;
  float scale_log2;
};

template <int D, bool kBf16>
__global__ void __launch_bounds__(128) decode_row_kernel(const Args a) {
  constexpr int kPer = D / 32;
  __shared__ float m_sh[4], l_sh[4], o_sh[4][D];
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int len = a.c.seqlens[b];
  if (len < 0 || len > a.c.max_len) {
    if (threadIdx.x == 0 && a.c.status) atomicOr(a.c.status, FA8_DEVERR_VARLEN_RANGE);
    return;
  }
  const int hk = h / (a.heads / a.c.heads_kv);
  const int n = len - a.seqlen_q + i + 1;  // keys this query sees
  float q[kPer], o[kPer];
  const char* qp = a.q + 2 * (b * a.q_sb + h * a.q_sh + i * a.q_ss + lane * kPer);
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    q[e] = (kBf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(qp)[e])
                  : __half2float(reinterpret_cast<const __half*>(qp)[e])) * a.scale_log2;
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int t = warp; t < n; t += 4) {
    const long long row = t < a.prefix_len ? 0 : b;
    const int page = a.c.table[row * a.c.table_stride + t / a.c.page_size];
    const int slot = t % a.c.page_size;
    float s = NAN, fv = NAN, v[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = 0.f;
    if (page >= 0 && page < a.c.num_pages) {
      const uint8_t* kp = a.c.k + page * a.c.k_sp + hk * a.c.k_sh + slot * a.c.k_ss + lane * kPer;
      const uint8_t* vp = a.c.v + page * a.c.v_sp + hk * a.c.v_sh + slot * a.c.v_ss + lane * kPer;
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < kPer; e += 2) {
        const uint32_t k2 = ptx::cvt_e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(kp + e));
        const uint32_t v2 = ptx::cvt_e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(vp + e));
        const float2 kf = __half22float2(*reinterpret_cast<const __half2*>(&k2));
        const float2 vf = __half22float2(*reinterpret_cast<const __half2*>(&v2));
        dot += q[e] * kf.x + q[e + 1] * kf.y;
        v[e] = vf.x;
        v[e + 1] = vf.y;
      }
#pragma unroll
      for (int w = 16; w; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
      s = dot * kv::exp_factor(a.c.k_exp[page * a.c.ke_sp + hk * a.c.ke_sh + slot]);
      fv = kv::exp_factor(a.c.v_exp[page * a.c.ve_sp + hk * a.c.ve_sh + slot]);
    } else if (lane == 0 && a.c.status) {
      atomicOr(a.c.status, FA8_DEVERR_PAGE_RANGE);
    }
    const float m_new = fmaxf(m, s);
    const float keep = exp2f(m - m_new), p = exp2f(s - m_new);
    l = l * keep + p;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = o[e] * keep + p * fv * v[e];
    m = m_new;
  }
  if (lane == 0) {
    m_sh[warp] = m;
    l_sh[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) o_sh[warp][lane * kPer + e] = o[e];
  __syncthreads();
  const float top = fmaxf(fmaxf(m_sh[0], m_sh[1]), fmaxf(m_sh[2], m_sh[3]));
  float sum = 0.f, w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    w[k] = m_sh[k] == -INFINITY && l_sh[k] == 0.f ? 0.f : exp2f(m_sh[k] - top);
    sum += w[k] * l_sh[k];
  }
  if (threadIdx.x < D) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) x += w[k] * o_sh[k][threadIdx.x];
    x = n > 0 ? x / sum : 0.f;
    const long long at = b * a.o_sb + h * a.o_sh + i * a.o_ss + threadIdx.x;
    if (kBf16)
      reinterpret_cast<__nv_bfloat16*>(a.o)[at] = __float2bfloat16(x);
    else
      reinterpret_cast<__half*>(a.o)[at] = __float2half(x);
  }
  if (threadIdx.x == 0 && a.lse)
    a.lse[((long long)b * a.heads + h) * a.seqlen_q + i] =
        n > 0 ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

// Host checks; *empty if there is nothing to compute.
int check(const fa8_decode_params* p, bool* empty) {
  *empty = true;
  if (!p) return fa8_note_error(FA8_ERR_INVALID_ARG, "params is NULL");
  if (p->heads < 0 || p->seqlen_q < 0 || p->cache.batch < 0 || p->prefix_len < 0)
    return fa8_note_error(FA8_ERR_INVALID_ARG, "fa8_decode: negative size");
  if (p->dtype != FA8_DT_F16 && p->dtype != FA8_DT_BF16)
    return fa8_note_error(FA8_ERR_INVALID_ARG, "fa8_decode: dtype must be FA8_DT_F16 or FA8_DT_BF16");
  if (p->cache.batch == 0 || p->heads == 0 || p->seqlen_q == 0) return FA8_OK;
  const int st = kv::check_cache(p->cache);
  if (st) return st;
  if (p->heads % p->cache.heads_kv != 0)
    return fa8_note_error(FA8_ERR_UNSUPPORTED, "fa8_decode: heads must be a multiple of heads_kv");
  if (p->heads > 65535 || p->seqlen_q > 65535 ||
      p->cache.batch * p->heads * p->seqlen_q > (1ll << 30))
    return fa8_note_error(FA8_ERR_UNSUPPORTED, "fa8_decode: too many query rows");
  if (p->prefix_len > p->cache.max_pages * p->cache.page_size)
    return fa8_note_error(FA8_ERR_INVALID_ARG, "fa8_decode: prefix_len does not fit the page table");
  if (!(p->softmax_scale > 0.f) || !std::isfinite(p->softmax_scale))
    return fa8_note_error(FA8_ERR_INVALID_ARG, "fa8_decode: softmax_scale must be positive and finite");
  if (!p->q || !p->o) return fa8_note_error(FA8_ERR_INVALID_ARG, "fa8_decode: null q or o");
  if ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->o)) & 15)
    return fa8_note_error(FA8_ERR_ALIGNMENT, "fa8_decode: q and o must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(p->lse) & 3)
    return fa8_note_error(FA8_ERR_ALIGNMENT, "fa8_decode: lse must be 4-byte aligned");
  for (int64_t s : {p->q_stride_b, p->q_stride_h, p->q_stride_s, p->o_stride_b, p->o_stride_h,
                    p->o_stride_s})
    if (s < 0 || s % 8 != 0)
      return fa8_note_error(FA8_ERR_ALIGNMENT,
                            "fa8_decode: strides of q and o must be multiples of 8 elements");
  *empty = false;
  return FA8_OK;
}

}  // namespace dec
}  // namespace fa8

extern "C" {

void fa8_decode_params_init(fa8_decode_params* p, int64_t num_pages, int64_t heads_kv,
                            int64_t page_size, int64_t head_dim, int64_t batch,
                            int64_t max_pages, int64_t heads, int64_t seqlen_q) {
  *p = fa8_decode_params();
  fa8_kv_cache_init(&p->cache, num_pages, heads_kv, page_size, head_dim, batch, max_pages);
  p->heads = heads;
  p->seqlen_q = seqlen_q;
  p->q_stride_s = p->o_stride_s = head_dim;
  p->q_stride_h = p->o_stride_h = seqlen_q * head_dim;
  p->q_stride_b = p->o_stride_b = heads * seqlen_q * head_dim;
  p->softmax_scale = head_dim > 0 ? 1.0f / sqrtf((float)head_dim) : 1.0f;
  p->dtype = FA8_DT_F16;
}

int64_t fa8_decode_workspace_size(const fa8_decode_params* p) {
  (void)p;
  return 0;
}

int fa8_decode(const fa8_decode_params* p, void* workspace, int64_t workspace_bytes, void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  bool empty;
  int st = fa8::dec::check(p, &empty);
  if (st || empty) return st;
  st = fa8::kv::check_device();
  if (st) return st;
  fa8::dec::Args a;
  a.c = fa8::kv::view_of(p->cache);
  a.q = static_cast<const char*>(p->q);
  a.o = static_cast<char*>(p->o);
  a.lse = p->lse;
  a.heads = (int)p->heads;
  a.seqlen_q = (int)p->seqlen_q;
  a.prefix_len = (int)p->prefix_len;
  a.q_sb = p->q_stride_b;
  a.q_sh = p->q_stride_h;
  a.q_ss = p->q_stride_s;
  a.o_sb = p->o_stride_b;
  a.o_sh = p->o_stride_h;
  a.o_ss = p->o_stride_s;
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  const dim3 grid((unsigned)p->seqlen_q, (unsigned)p->heads, (unsigned)p->cache.batch);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf16 = p->dtype == FA8_DT_BF16;
  auto launch = [&](auto kernel) { kernel<<<grid, 128, 0, s>>>(a); };
  if (p->cache.head_dim == 128)
    launch(bf16 ? fa8::dec::decode_row_kernel<128, true> : fa8::dec::decode_row_kernel<128, false>);
  else
    launch(bf16 ? fa8::dec::decode_row_kernel<64, true> : fa8::dec::decode_row_kernel<64, false>);
  fa8_note_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FA8_OK : fa8_note_cuda_error(e, "decode kernel launch");
}

}  // extern "C"
