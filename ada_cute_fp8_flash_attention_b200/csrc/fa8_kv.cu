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
// the maximum is taken by shuffles without shared memory. The maximum is taken
// on the magnitude bits (16-bit integers order as the values do, with
// infinities and NaN on top), two elements of a packed max at a time.
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
  int total;                // tokens of the call
  int tokens;               // per sequence, without cu
  int per_block;            // tokens of a block
  Divisor by_heads;         // (heads_kv)
  long long k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;
};

// Blocks of the row kernel that the GPU holds at once (148 SMs, 8 each).
constexpr int64_t kOneWave = 148 * 8;
constexpr int kCopyThreads = 256;
constexpr int kMostTokens = 16;  // of a block

// Where a token lives on either side: element offsets of its head 0 in k and
// v, byte offsets in the cache. page -1: outside the cache; -2: no such token.
struct Place {
  long long k, v;
  long long ck, cv, ek, ev;
  int page;
};

__device__ __forceinline__ Place place_of(const CopyArgs& a, int tok) {
  Place p;
  p.page = -2;
  if (tok >= a.total) return p;
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
    n = (int)((unsigned)c1 - (unsigned)c0);
    back = c1 - tok;
    p.k = tok * a.k_ss;
    p.v = tok * a.v_ss;
  } else {
    b = tok / a.tokens;
    const int i = tok - b * a.tokens;
    n = a.tokens;
    back = n - i;
    p.k = b * a.k_sb + i * a.k_ss;
    p.v = b * a.v_sb + i * a.v_ss;
  }
  const int len = __ldg(a.c.seqlens + b);
  if (len > a.c.max_len || len < n || n < 0) {  // (n wraps if cu[0] is far below 0)
    if (a.c.status) atomicOr(a.c.status, FA8_DEVERR_VARLEN_RANGE);
    return p;
  }
  const int pos = len - back;
  const int col = pos / a.c.page_size, slot = pos - col * a.c.page_size;
  p.page = __ldg(a.c.table + b * a.c.table_stride + col);
  if (p.page < 0 || p.page >= a.c.num_pages) {
    if (a.c.status) atomicOr(a.c.status, FA8_DEVERR_PAGE_RANGE);
    p.page = -1;
    return p;
  }
  p.ck = p.page * a.c.k_sp + slot * a.c.k_ss;
  p.cv = p.page * a.c.v_sp + slot * a.c.v_ss;
  p.ek = p.page * a.c.ke_sp + slot;
  p.ev = p.page * a.c.ve_sp + slot;
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

// One row of K and of V per group of lanes, each finding its own place: for
// calls whose rows fit the GPU at once, where this is the shortest way.
template <int D, bool kBf16, bool kWrite>
__global__ void __launch_bounds__(kCopyThreads) kv_copy_row_kernel(const CopyArgs a) {
  constexpr int kLanes = D / 8;
  const int lane = threadIdx.x % kLanes;
  const int row = (blockIdx.x * kCopyThreads + threadIdx.x) / kLanes;
  const int tok = a.by_heads.div(row);
  const int head = row - tok * a.c.heads_kv;
  const Place p = place_of(a, tok);
  const CacheView& c = a.c;
  if constexpr (kWrite) {
    uint4 xk = make_uint4(0, 0, 0, 0), xv = xk;
    if (p.page >= 0) {
      xk = __ldcs(reinterpret_cast<const uint4*>(a.k + 2 * (p.k + head * a.k_sh)) + lane);
      xv = __ldcs(reinterpret_cast<const uint4*>(a.v + 2 * (p.v + head * a.v_sh)) + lane);
    }
    int bk, bv;  // every lane of the warp takes part in the shuffles
    const uint2 ck = quantise<kLanes, kBf16>(xk, bk);
    const uint2 cv = quantise<kLanes, kBf16>(xv, bv);
    if (p.page < 0) return;
    reinterpret_cast<uint2*>(c.k + p.ck + head * c.k_sh)[lane] = ck;
    reinterpret_cast<uint2*>(c.v + p.cv + head * c.v_sh)[lane] = cv;
    if (lane == 0) {
      c.k_exp[p.ek + head * c.ke_sh] = (uint8_t)bk;
      c.v_exp[p.ev + head * c.ve_sh] = (uint8_t)bv;
    }
  } else {
    if (p.page == -2) return;
    uint2 ck = make_uint2(0, 0), cv = ck;
    int bk = kExpNan, bv = kExpNan;
    if (p.page >= 0) {
      ck = reinterpret_cast<const uint2*>(c.k + p.ck + head * c.k_sh)[lane];
      cv = reinterpret_cast<const uint2*>(c.v + p.cv + head * c.v_sh)[lane];
      bk = c.k_exp[p.ek + head * c.ke_sh];
      bv = c.v_exp[p.ev + head * c.ve_sh];
    }
    reinterpret_cast<uint4*>(a.k + 2 * (p.k + head * a.k_sh))[lane] = dequantise<kBf16>(ck, bk);
    reinterpret_cast<uint4*>(a.v + 2 * (p.v + head * a.v_sh))[lane] = dequantise<kBf16>(cv, bv);
  }
}

// A block moves `per_block` tokens, all heads: row r of it is head r % heads of
// token r / heads. The tokens' places are found once, by one thread each; then
// every thread keeps the rows of a batch of K and V in flight together.
template <int D, bool kBf16, bool kWrite>
__global__ void __launch_bounds__(kCopyThreads, kWrite ? 8 : 1) kv_copy_kernel(const CopyArgs a) {
  constexpr int kLanes = D / 8, kGroups = kCopyThreads / kLanes;
  // Rows of K and of V that a thread has asked for: 2, 4, 8 took 88, 91, 119 us
  // (write) and 70, 68, 83 us (read) for 65000 and 55000 tokens of 8 heads; with
  // eight blocks an SM the write takes 84, the read 80.
  constexpr int kRowsInFlight = kWrite ? 2 : 4;
  __shared__ Place places[kMostTokens];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  if (threadIdx.x < a.per_block)
    places[threadIdx.x] = place_of(a, blockIdx.x * a.per_block + threadIdx.x);
  __syncthreads();
  const CacheView& c = a.c;
  const int rows = a.per_block * c.heads_kv;
#pragma unroll 1
  for (int base = 0; base < rows; base += kGroups * kRowsInFlight) {
    const int r0 = base + group;
    if constexpr (kWrite) {
      uint4 xk[kRowsInFlight], xv[kRowsInFlight];
      int tok[kRowsInFlight], head[kRowsInFlight];
#pragma unroll
      for (int u = 0; u < kRowsInFlight; ++u) {
        const int r = r0 + u * kGroups;
        tok[u] = a.by_heads.div(r);
        head[u] = r - tok[u] * c.heads_kv;
        xk[u] = xv[u] = make_uint4(0, 0, 0, 0);
        if (r >= rows || places[tok[u]].page < 0) {
          tok[u] = -1;
          continue;
        }
        const Place& p = places[tok[u]];
        xk[u] = __ldcs(reinterpret_cast<const uint4*>(a.k + 2 * (p.k + head[u] * a.k_sh)) + lane);
        xv[u] = __ldcs(reinterpret_cast<const uint4*>(a.v + 2 * (p.v + head[u] * a.v_sh)) + lane);
      }
#pragma unroll
      for (int u = 0; u < kRowsInFlight; ++u) {
        // Every lane of the warp takes part in the shuffles.
        int bk, bv;
        const uint2 ck = quantise<kLanes, kBf16>(xk[u], bk);
        const uint2 cv = quantise<kLanes, kBf16>(xv[u], bv);
        if (tok[u] < 0) continue;
        const Place& p = places[tok[u]];
        reinterpret_cast<uint2*>(c.k + p.ck + head[u] * c.k_sh)[lane] = ck;
        reinterpret_cast<uint2*>(c.v + p.cv + head[u] * c.v_sh)[lane] = cv;
        if (lane == 0) {
          c.k_exp[p.ek + head[u] * c.ke_sh] = (uint8_t)bk;
          c.v_exp[p.ev + head[u] * c.ve_sh] = (uint8_t)bv;
        }
      }
    } else {
      uint2 ck[kRowsInFlight], cv[kRowsInFlight];
      int bk[kRowsInFlight], bv[kRowsInFlight], tok[kRowsInFlight], head[kRowsInFlight];
#pragma unroll
      for (int u = 0; u < kRowsInFlight; ++u) {
        const int r = r0 + u * kGroups;
        tok[u] = a.by_heads.div(r);
        head[u] = r - tok[u] * c.heads_kv;
        ck[u] = cv[u] = make_uint2(0, 0);
        bk[u] = bv[u] = kExpNan;
        if (r >= rows || places[tok[u]].page == -2) {
          tok[u] = -1;
          continue;
        }
        const Place& p = places[tok[u]];
        if (p.page < 0) continue;
        ck[u] = __ldcs(reinterpret_cast<const uint2*>(c.k + p.ck + head[u] * c.k_sh) + lane);
        cv[u] = __ldcs(reinterpret_cast<const uint2*>(c.v + p.cv + head[u] * c.v_sh) + lane);
        bk[u] = c.k_exp[p.ek + head[u] * c.ke_sh];
        bv[u] = c.v_exp[p.ev + head[u] * c.ve_sh];
      }
#pragma unroll
      for (int u = 0; u < kRowsInFlight; ++u) {
        if (tok[u] < 0) continue;
        const Place& p = places[tok[u]];
        __stcs(reinterpret_cast<uint4*>(a.k + 2 * (p.k + head[u] * a.k_sh)) + lane,
               dequantise<kBf16>(ck[u], bk[u]));
        __stcs(reinterpret_cast<uint4*>(a.v + 2 * (p.v + head[u] * a.v_sh)) + lane,
               dequantise<kBf16>(cv[u], bv[u]));
      }
    }
  }
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
  const int64_t total = p->tokens * (p->cu_seqlens ? 1 : p->cache.batch);
  if (total > (1ll << 30))
    return fa8_note_error(FA8_ERR_UNSUPPORTED, "cache copy: too many tokens");
  a.tokens = (int)p->tokens;
  a.total = (int)total;
  const int64_t heads = p->cache.heads_kv;
  a.by_heads = Divisor::of((int)heads);
  a.k_sb = p->k_stride_b;
  a.k_sh = p->k_stride_h;
  a.k_ss = p->k_stride_s;
  a.v_sb = p->v_stride_b;
  a.v_sh = p->v_stride_h;
  a.v_ss = p->v_stride_s;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf16 = p->dtype == FA8_DT_BF16;
  const int64_t groups = kCopyThreads / (p->cache.head_dim / 8);  // rows of a block at a time
  const bool by_rows = total * heads <= groups * kOneWave;
  a.per_block = kMostTokens;
  const unsigned blocks =
      by_rows ? (unsigned)((total * heads + groups - 1) / groups)
              : (unsigned)((total + a.per_block - 1) / a.per_block);
  auto launch = [&](auto rows, auto tokens) {
    (by_rows ? rows : tokens)<<<blocks, kCopyThreads, 0, s>>>(a);
  };
  if (p->cache.head_dim == 128)
    launch(bf16 ? kv_copy_row_kernel<128, true, kWrite> : kv_copy_row_kernel<128, false, kWrite>,
           bf16 ? kv_copy_kernel<128, true, kWrite> : kv_copy_kernel<128, false, kWrite>);
  else
    launch(bf16 ? kv_copy_row_kernel<64, true, kWrite> : kv_copy_row_kernel<64, false, kWrite>,
           bf16 ? kv_copy_kernel<64, true, kWrite> : kv_copy_kernel<64, false, kWrite>);
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
