// fa8_kv.cu — a paged e4m3 key/value cache: quantising tokens into it
// (fa8_kv_write) and reading them back (fa8_kv_read). No counterpart in the
// reference.
//
// Write, per row x of D elements (one token, K/V head, K or V):
//   a = max |x|,  e = least integer >= -63 with a <= 448 * 2^e (0 if a = 0),
//   byte = e + 127,  code = rn_e4m3(x * 2^-e).
// Read: y = rn(code * 2^e) in fp16 or bf16, saturating.
//
// Both are bound by HBM: 2 D bytes on one side, D + 1 on the other, a handful
// of operations each element. D / 8 lanes hold one row, 16 bytes a lane, so
// that a half warp (D = 128) moves 256 contiguous bytes of a row at once and
// the maximum is taken by shuffles without shared memory; each thread moves
// its piece of K and of V, two independent loads in flight. The maximum is
// taken on the magnitude bits (16-bit integers order as the values do, with
// infinities and NaN on top), two lanes of a packed max at a time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "fa8_kv.cuh"
#include "sm100_ptx.cuh"

namespace fa8 {
namespace kv {

int check_cache(const fa8_kv_cache& c) {
  if (c.head_dim != 64 && c.head_dim != 128)
    return fa8_note_error(FA8_ERR_UNSUPPORTED, "cache: head_dim must be 64 or 128");
  if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 &&
      (c.page_size <= 0 || c.page_size % 128 != 0))
    return fa8_note_error(FA8_ERR_UNSUPPORTED,
                          "cache: page_size must be 16, 32, 64 or a multiple of 128");
  if (c.num_pages < 0 || c.heads_kv <= 0 || c.batch < 0 || c.max_pages < 0)
    return fa8_note_error(FA8_ERR_INVALID_ARG, "cache: negative size or no K/V head");
  if (c.num_pages > 0x7fffffff || c.heads_kv > 65535 || c.batch > 65535 ||
      c.page_size > (1 << 20) || c.max_pages > (1 << 30) / c.page_size)
    return fa8_note_error(FA8_ERR_UNSUPPORTED, "cache: size exceeds the supported index range");
  if (!c.seqlens || (c.max_pages > 0 && !c.page_table))
    return fa8_note_error(FA8_ERR_INVALID_ARG, "cache: null page_table or seqlens");
  if (c.num_pages > 0 && (!c.k || !c.v || !c.k_exp || !c.v_exp))
    return fa8_note_error(FA8_ERR_INVALID_ARG, "cache: null codes or exponents");
  if (c.max_pages > 0 && c.table_stride < 0)
    return fa8_note_error(FA8_ERR_INVALID_ARG, "cache: negative table_stride");
  if ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15)
    return fa8_note_error(FA8_ERR_ALIGNMENT, "cache: codes must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(c.page_table) | reinterpret_cast<uintptr_t>(c.seqlens) |
       reinterpret_cast<uintptr_t>(c.status)) & 3)
    return fa8_note_error(FA8_ERR_ALIGNMENT, "cache: int32 arrays must be 4-byte aligned");
  for (int64_t s : {c.k_stride_p, c.k_stride_h, c.k_stride_s, c.v_stride_p, c.v_stride_h,
                    c.v_stride_s})
    if (s <= 0 || s % 16 != 0)
      return fa8_note_error(FA8_ERR_ALIGNMENT,
                            "cache: strides of the codes must be positive multiples of 16");
  if (c.k_stride_s < c.head_dim || c.v_stride_s < c.head_dim)
    return fa8_note_error(FA8_ERR_INVALID_ARG, "cache: slots overlap (stride_s < head_dim)");
  for (int64_t s : {c.k_exp_stride_p, c.k_exp_stride_h, c.v_exp_stride_p, c.v_exp_stride_h})
    if (s <= 0)
      return fa8_note_error(FA8_ERR_INVALID_ARG, "cache: exponent strides must be positive");
  // The attention reads them 16 at a time.
  if (((reinterpret_cast<uintptr_t>(c.k_exp) | reinterpret_cast<uintptr_t>(c.v_exp)) & 15) ||
      ((c.k_exp_stride_p | c.k_exp_stride_h | c.v_exp_stride_p | c.v_exp_stride_h) & 15))
    return fa8_note_error(FA8_ERR_ALIGNMENT,
                          "cache: exponents must be 16-byte aligned, their strides multiples of 16");
  return FA8_OK;
}

int check_device() {
  int dev = 0, major = 0, minor = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
  if (e != cudaSuccess) return fa8_note_cuda_error(e, "cudaDeviceGetAttribute");
  if (major != 10 || minor != 0)
    return fa8_note_error(FA8_ERR_NO_DEVICE, "the current device is not sm_100 (B200)");
  return FA8_OK;
}

namespace {

struct CopyArgs {
  CacheView c;
  char* k;
  char* v;
  const int* cu;
  long long rows;           // (token, head) pairs in all
  int tokens;               // packed rows, or tokens per sequence
  long long k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;
};

struct Place {
  long long src_k, src_v;   // element offsets of the row in k and v
  int page, slot, head;
  bool ok;
};

// Where row `idx` = (token, head) lives on either side. Lanes of one row get
// the same answer; only `lead` reports what is refused.
__device__ __forceinline__ Place place_of(const CopyArgs& a, long long idx, bool lead) {
  Place p;
  p.ok = false;
  p.page = p.slot = 0;
  p.src_k = p.src_v = 0;
  const long long tok = idx / a.c.heads_kv;
  p.head = (int)(idx - tok * a.c.heads_kv);
  int b, back;  // back: distance from the sequence's end, 1 = its last token
  int n;        // tokens of this sequence in the call
  if (a.cu) {
    // The last b with cu[b] <= tok.
    int lo = 0, hi = a.c.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(a.cu + mid) <= tok) lo = mid; else hi = mid;
    }
    b = lo;
    const int c0 = __ldg(a.cu + b), c1 = __ldg(a.cu + b + 1);
    if (tok < c0 || tok >= c1) return p;  // before the first or behind the last sequence
    n = c1 - c0;
    back = c1 - (int)tok;
    p.src_k = tok * a.k_ss + p.head * a.k_sh;
    p.src_v = tok * a.v_ss + p.head * a.v_sh;
  } else {
    b = (int)(tok / a.tokens);
    const int i = (int)(tok - (long long)b * a.tokens);
    n = a.tokens;
    back = n - i;
    p.src_k = b * a.k_sb + p.head * a.k_sh + i * a.k_ss;
    p.src_v = b * a.v_sb + p.head * a.v_sh + i * a.v_ss;
  }
  const int len = __ldg(a.c.seqlens + b);
  if (len > a.c.max_len || len < n) {
    if (lead && a.c.status) atomicOr(a.c.status, FA8_DEVERR_VARLEN_RANGE);
    return p;
  }
  const int pos = len - back;
  const int col = pos / a.c.page_size;
  p.slot = pos - col * a.c.page_size;
  p.page = __ldg(a.c.table + b * a.c.table_stride + col);
  if (p.page < 0 || p.page >= a.c.num_pages) {
    if (lead && a.c.status) atomicOr(a.c.status, FA8_DEVERR_PAGE_RANGE);
    p.page = -1;
  }
  p.ok = true;
  return p;
}

template <bool kBf16>
__device__ __forceinline__ float2 to_float2(uint32_t w) {
  if constexpr (kBf16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}

// Quantise one row spread over `kLanes` lanes, 8 elements each.
template <int kLanes, bool kBf16>
__device__ __forceinline__ uint2 quantise(uint4 x, int& byte) {
  uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                        __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
  m = max(m & 0xffffu, m >> 16);
#pragma unroll
  for (int o = kLanes / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m >= (kBf16 ? 0x7f80u : 0x7c00u)) {
    byte = kExpNan;
    return make_uint2(0u, 0u);
  }
  const uint32_t bits = __float_as_uint(to_float2<kBf16>(m).x);
  // a = 1.f * 2^(E - 127) against 448 = 1.75 * 2^8.
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = m == 0 ? 0 : max(e, kMinExp);
  byte = e + kExpBias;
  const float f = __uint_as_float((uint32_t)(127 - e) << 23);
  const float2 p0 = to_float2<kBf16>(x.x), p1 = to_float2<kBf16>(x.y), p2 = to_float2<kBf16>(x.z),
               p3 = to_float2<kBf16>(x.w);
  return make_uint2(ptx::cvt_e4m3x4(p0.x * f, p0.y * f, p1.x * f, p1.y * f),
                    ptx::cvt_e4m3x4(p2.x * f, p2.y * f, p3.x * f, p3.y * f));
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack_sat(float lo, float hi) {
  uint32_t r;
  if constexpr (kBf16)
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <bool kBf16>
__device__ __forceinline__ uint4 dequantise(uint2 c, int byte) {
  const float f = exp_factor(byte);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t word = i < 2 ? c.x : c.y;
    const uint32_t h = ptx::cvt_e4m3x2_to_f16x2((uint16_t)(i & 1 ? word >> 16 : word & 0xffffu));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
    w[i] = pack_sat<kBf16>(x.x * f, x.y * f);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int kCopyThreads = 256;

template <int D, bool kBf16>
__global__ void __launch_bounds__(kCopyThreads) kv_write_kernel(const CopyArgs a) {
  constexpr int kLanes = D / 8;
  const long long idx = (blockIdx.x * (long long)kCopyThreads + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  Place p;
  p.ok = false;
  if (idx < a.rows) p = place_of(a, idx, lane == 0);
  const bool go = p.ok && p.page >= 0;
  uint4 xk = make_uint4(0, 0, 0, 0), xv = xk;
  if (go) {
    xk = __ldcs(reinterpret_cast<const uint4*>(a.k + 2 * p.src_k) + lane);
    xv = __ldcs(reinterpret_cast<const uint4*>(a.v + 2 * p.src_v) + lane);
  }
  // Every lane of the warp takes part in the shuffles.
  int bk, bv;
  const uint2 ck = quantise<kLanes, kBf16>(xk, bk);
  const uint2 cv = quantise<kLanes, kBf16>(xv, bv);
  if (!go) return;
  const CacheView& c = a.c;
  reinterpret_cast<uint2*>(c.k + p.page * c.k_sp + p.head * c.k_sh + p.slot * c.k_ss)[lane] = ck;
  reinterpret_cast<uint2*>(c.v + p.page * c.v_sp + p.head * c.v_sh + p.slot * c.v_ss)[lane] = cv;
  if (lane == 0) {
    c.k_exp[p.page * c.ke_sp + p.head * c.ke_sh + p.slot] = (uint8_t)bk;
    c.v_exp[p.page * c.ve_sp + p.head * c.ve_sh + p.slot] = (uint8_t)bv;
  }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kCopyThreads) kv_read_kernel(const CopyArgs a) {
  constexpr int kLanes = D / 8;
  const long long idx = (blockIdx.x * (long long)kCopyThreads + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  if (idx >= a.rows) return;
  const Place p = place_of(a, idx, lane == 0);
  if (!p.ok) return;
  const CacheView& c = a.c;
  uint2 ck = make_uint2(0, 0), cv = ck;
  int bk = kExpNan, bv = kExpNan;
  if (p.page >= 0) {
    ck = reinterpret_cast<const uint2*>(c.k + p.page * c.k_sp + p.head * c.k_sh +
                                        p.slot * c.k_ss)[lane];
    cv = reinterpret_cast<const uint2*>(c.v + p.page * c.v_sp + p.head * c.v_sh +
                                        p.slot * c.v_ss)[lane];
    bk = c.k_exp[p.page * c.ke_sp + p.head * c.ke_sh + p.slot];
    bv = c.v_exp[p.page * c.ve_sp + p.head * c.ve_sh + p.slot];
  }
  __stcs(reinterpret_cast<uint4*>(a.k + 2 * p.src_k) + lane, dequantise<kBf16>(ck, bk));
  __stcs(reinterpret_cast<uint4*>(a.v + 2 * p.src_v) + lane, dequantise<kBf16>(cv, bv));
}

int check_copy(const fa8_kv_copy_params* p, bool* empty) {
  *empty = true;
  if (!p) return fa8_note_error(FA8_ERR_INVALID_ARG, "params is NULL");
  if (p->tokens < 0 || p->cache.batch < 0)
    return fa8_note_error(FA8_ERR_INVALID_ARG, "cache copy: negative size");
  if (p->dtype != FA8_DT_F16 && p->dtype != FA8_DT_BF16)
    return fa8_note_error(FA8_ERR_INVALID_ARG, "cache copy: dtype must be FA8_DT_F16 or FA8_DT_BF16");
  if (p->cache.batch == 0 || p->tokens == 0) return FA8_OK;
  const int st = check_cache(p->cache);
  if (st) return st;
  if (!p->k || !p->v) return fa8_note_error(FA8_ERR_INVALID_ARG, "cache copy: null k or v");
  if (p->tokens > (1ll << 30))
    return fa8_note_error(FA8_ERR_UNSUPPORTED, "cache copy: too many tokens");
  if ((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15)
    return fa8_note_error(FA8_ERR_ALIGNMENT, "cache copy: k and v must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(p->cu_seqlens) & 3)
    return fa8_note_error(FA8_ERR_ALIGNMENT, "cache copy: cu_seqlens must be 4-byte aligned");
  for (int64_t s : {p->k_stride_h, p->k_stride_s, p->v_stride_h, p->v_stride_s,
                    p->cu_seqlens ? 0 : p->k_stride_b, p->cu_seqlens ? 0 : p->v_stride_b})
    if (s < 0 || s % 8 != 0)
      return fa8_note_error(FA8_ERR_ALIGNMENT,
                            "cache copy: strides of k and v must be multiples of 8 elements");
  *empty = false;
  return FA8_OK;
}

template <bool kWrite>
int copy(const fa8_kv_copy_params* p, void* stream) {
  bool empty;
  int st = check_copy(p, &empty);
  if (st || empty) return st;
  st = check_device();
  if (st) return st;
  CopyArgs a;
  a.c = view_of(p->cache);
  a.k = static_cast<char*>(p->k);
  a.v = static_cast<char*>(p->v);
  a.cu = p->cu_seqlens;
  a.tokens = (int)p->tokens;
  a.rows = p->tokens * p->cache.heads_kv * (p->cu_seqlens ? 1 : p->cache.batch);
  a.k_sb = p->k_stride_b;
  a.k_sh = p->k_stride_h;
  a.k_ss = p->k_stride_s;
  a.v_sb = p->v_stride_b;
  a.v_sh = p->v_stride_h;
  a.v_ss = p->v_stride_s;
  const int per_block = kCopyThreads / (int)(p->cache.head_dim / 8);
  const int64_t blocks = (a.rows + per_block - 1) / per_block;
  if (blocks > 0x7fffffff)
    return fa8_note_error(FA8_ERR_UNSUPPORTED, "cache copy: too many rows");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf16 = p->dtype == FA8_DT_BF16;
  auto launch = [&](auto kernel) { kernel<<<(unsigned)blocks, kCopyThreads, 0, s>>>(a); };
  if constexpr (kWrite) {
    if (p->cache.head_dim == 128)
      launch(bf16 ? kv_write_kernel<128, true> : kv_write_kernel<128, false>);
    else
      launch(bf16 ? kv_write_kernel<64, true> : kv_write_kernel<64, false>);
  } else {
    if (p->cache.head_dim == 128)
      launch(bf16 ? kv_read_kernel<128, true> : kv_read_kernel<128, false>);
    else
      launch(bf16 ? kv_read_kernel<64, true> : kv_read_kernel<64, false>);
  }
  fa8_note_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FA8_OK : fa8_note_cuda_error(e, "cache copy kernel launch");
}

}  // namespace
}  // namespace kv
}  // namespace fa8

extern "C" {

void fa8_kv_cache_init(fa8_kv_cache* c, int64_t num_pages, int64_t heads_kv, int64_t page_size,
                       int64_t head_dim, int64_t batch, int64_t max_pages) {
  *c = fa8_kv_cache();
  c->num_pages = num_pages;
  c->heads_kv = heads_kv;
  c->page_size = page_size;
  c->head_dim = head_dim;
  c->k_stride_s = c->v_stride_s = head_dim;
  c->k_stride_h = c->v_stride_h = page_size * head_dim;
  c->k_stride_p = c->v_stride_p = heads_kv * page_size * head_dim;
  c->k_exp_stride_h = c->v_exp_stride_h = page_size;
  c->k_exp_stride_p = c->v_exp_stride_p = heads_kv * page_size;
  c->batch = batch;
  c->table_stride = max_pages;
  c->max_pages = max_pages;
}

int fa8_kv_write(const fa8_kv_copy_params* p, void* stream) {
  return fa8::kv::copy<true>(p, stream);
}

int fa8_kv_read(const fa8_kv_copy_params* p, void* stream) {
  return fa8::kv::copy<false>(p, stream);
}

}  // extern "C"
