// fa8_kv.cuh — what the cache kernels (fa8_kv.cu) and the attention over the
// cache (fa8_decode.cu) share: the device view of a paged e4m3 key/value
// cache and the host checks of one.
//
// A row (one token, one K/V head, K or V) is D e4m3 codes and one exponent
// byte: value = code * 2^(byte - 127). The factor is a power of two because
// e4m3 is a floating-point format: a finer factor would move values within
// their binade, which changes no relative error; a power of two costs at most
// one of the format's 18 binades, one byte instead of four, and makes x * 2^-e
// and code * 2^e exact, so that a value is rounded once on its way in.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/fa8.h"

int fa8_note_error(int status, const char* msg);
int fa8_note_cuda_error(cudaError_t e, const char* where);
void fa8_note_launch();

namespace fa8 {
namespace kv {

// x / d for 0 <= x < 2^31 by one multiplication (the division by an invariant of
// Granlund and Montgomery, PLDI 1994): with 2^shift the least power of two that is
// not below d and mul = floor(2^32 (2^shift - d) / d) + 1, the quotient is
// (floor(mul x / 2^32) + x) / 2^shift; x below 2^31 keeps that sum in 32 bits.
struct Divisor {
  uint32_t mul, shift;
  int d;
  static Divisor of(int d) {
    Divisor v{0, 0, d};
    while ((1ll << v.shift) < d) ++v.shift;
    v.mul = (uint32_t)((((1ull << v.shift) - d) << 32) / d + 1);
    return v;
  }
  __device__ __forceinline__ int div(int x) const {
    return (int)((__umulhi((uint32_t)x, mul) + (uint32_t)x) >> shift);
  }
};

struct CacheView {
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_exp;
  uint8_t* v_exp;
  long long k_sp, k_sh, k_ss, v_sp, v_sh, v_ss;  // strides of the codes
  long long ke_sp, ke_sh, ve_sp, ve_sh;          // of the exponent bytes
  const int* table;
  long long table_stride;
  const int* seqlens;
  int* status;
  int num_pages, heads_kv, page_size, batch;
  int max_len;  // tokens that a table row can hold
};

constexpr int kExpNan = 255;   // byte of a row that held an infinity or a NaN
constexpr int kExpBias = 127;
// Least exponent of a written row: values below 2^-73, half the least subnormal
// code, become zero. (Attention takes any: see kWide in fa8_decode.cu.)
constexpr int kMinExp = -63;

__device__ __forceinline__ float exp_factor(int byte) {
  return __int_as_float(byte == kExpNan ? 0x7fc00000 : (byte == 0 ? 0x00400000 : byte << 23));
}

inline CacheView view_of(const fa8_kv_cache& c) {
  CacheView v;
  v.k = static_cast<uint8_t*>(c.k);
  v.v = static_cast<uint8_t*>(c.v);
  v.k_exp = c.k_exp;
  v.v_exp = c.v_exp;
  v.k_sp = c.k_stride_p;
  v.k_sh = c.k_stride_h;
  v.k_ss = c.k_stride_s;
  v.v_sp = c.v_stride_p;
  v.v_sh = c.v_stride_h;
  v.v_ss = c.v_stride_s;
  v.ke_sp = c.k_exp_stride_p;
  v.ke_sh = c.k_exp_stride_h;
  v.ve_sp = c.v_exp_stride_p;
  v.ve_sh = c.v_exp_stride_h;
  v.table = c.page_table;
  v.table_stride = c.table_stride;
  v.seqlens = c.seqlens;
  v.status = c.status;
  v.num_pages = (int)c.num_pages;
  v.heads_kv = (int)c.heads_kv;
  v.page_size = (int)c.page_size;
  v.batch = (int)c.batch;
  v.max_len = (int)(c.max_pages * c.page_size);
  return v;
}

// Host checks of a cache whose batch is not empty; FA8_OK or a noted error.
int check_cache(const fa8_kv_cache& c);
// FA8_OK if the current device is a B200.
int check_device();

}  // namespace kv
}  // namespace fa8
