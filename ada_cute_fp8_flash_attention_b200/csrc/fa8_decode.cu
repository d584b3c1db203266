// fa8_decode.cu — attention of the last few tokens of every sequence over a
// paged e4m3 cache (fa8_decode), optionally with a prefix that all sequences
// share. No counterpart in the reference.
//
//   s_j = scale * q . k_j,  o = sum_j exp(s_j) v_j / sum_j exp(s_j),
//   lse = ln sum_j exp(s_j),  over the keys j <= position of the query.
//
// What bounds it: a key costs 2 (D + 1) bytes of HBM and 4 D operations a
// query row. One row per K/V head is far below what tensor cores need to be
// busy, so the bytes bound it as long as the arithmetic beside the loads
// stays off the critical path. 6.5 TB/s are 23 bytes a clock and SM, a key
// (D = 128) every 11 clocks: converting K and V to 16 bits in registers (256
// values a key) would take most of the issue slots. So K and V are never
// converted: they go from HBM through TMA into shared memory and from there
// into tcgen05.mma kind::f8f6f4 as the e4m3 bytes they are, always as the
// 128-row operand A,
//   S^T = K Q^T  (128 keys x rows),   O^T += V^T P^T  (D x rows),
// with the few query rows along N, where small sizes are cheap. One thread
// then holds one key: its exponent bytes are two registers, its column of P
// one or a few 16-byte stores.
//
// Rows to 8 bits. tcgen05 wants Q and P in e4m3 too. A value x is held as
// terms x = t0 + t1 / 16 + t2 / 256, t0 = rn(x), t1 = rn(16 (x - t0)), ...;
// e4m3 has 4 significant bits and a rounding is off by half a step, so two
// terms hold 8 bits and three hold 11 or more: what bf16 and fp16 have. The
// terms are columns of their own (N is 2 or 3 times the rows) and are added
// up in fp32 with their weights. Q is held exactly (scaled by a power of two
// per row so that its largest magnitude is in [128, 256)); P is rounded once
// to 11 (fp16) or 8 (bf16) bits, as it would be for a 16-bit product.
//
// Softmax in base 2 with one running maximum per row, m = max(s + e), e the
// exponent of v_j: then p = 2^(s - m) enters the sum, and what goes to the
// product is 2^5 * 2^(e) * p <= 2^5 whatever the exponents are (times 2^3,
// the rise of the maximum below which nothing is rescaled). The sum is kept
// per thread, over its own keys, and joined at the end of a row's keys.
//
// Work. Key tiles of 128 of all (sequence, K/V head, tile of query rows) are
// numbered through; block c of G = min(blocks, U) takes those from U c / G to
// U (c + 1) / G,
// found from the lengths on the device by a scan: any mixture of lengths
// shares the GPU evenly and nothing is read on the host. A block that holds
// all of an item's keys writes the result; else it writes its unnormalised
// sums, and a second kernel, launched early and waiting on the device for the
// first, joins them (always the same shares: results repeat bit by bit).
//
// A shared prefix is one more set of items, whose rows are those of the whole
// batch: one launch for it, one for what is behind it, one that joins both.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <mutex>

#include "fa8_kv.cuh"
#include "sm100_ptx.cuh"

namespace fa8 {
namespace dec {

constexpr int kTileKeys = 128;
constexpr float kRise = 3.f;           // log2 of the rise of a maximum that is let be
constexpr float kPScale = 32.f;        // 2^5 p 2^e <= 2^(5 + kRise) < 448
constexpr float kTerm = 16.f;          // weight of a term over the next
constexpr long long kTimeout = 4000000000LL;
constexpr int kWaitHintNs = 20000;

// Where an item's result is, for the kernel that joins the prefix with what is
// behind it.
enum { kItemEmpty = 0, kItemFull = 1, kItemParts = 2 };

// D: head dimension. NT: e4m3 terms of Q and P (2 bf16, 3 fp16). RW: query
// rows of a softmax warpgroup. NWG: warpgroups, each with its own rows.
template <int D_, int NT_, int RW_, int NWG_>
struct Cfg {
  static constexpr int D = D_, NT = NT_, RW = RW_, NWG = NWG_;
  static constexpr int kRows = RW * NWG;
  static constexpr int kThreads = NWG * 128 + 64;
  static constexpr int kMmaWarp = NWG * 4, kLoadWarp = NWG * 4 + 1;
  static constexpr int kN = (NT * RW + 15) / 16 * 16;  // columns of the products
  static constexpr int kPitch = kN <= 64 ? 64 : 128;   // bytes of a key's row of P
  static constexpr int kSlotBytes = kTileKeys * D;     // a K or a V tile
  static constexpr int kQBytes = kN * D;               // per warpgroup
  static constexpr int kPBytes = kTileKeys * kPitch;
  static constexpr uint32_t kTmemUsed = 2u * kN * NWG;
  static constexpr uint32_t kTmemCols =
      kTmemUsed <= 32 ? 32 : kTmemUsed <= 64 ? 64 : kTmemUsed <= 128 ? 128 : kTmemUsed <= 256 ? 256 : 512;
  static constexpr int kCtas = NWG > 1 ? 1 : (D == 64 && RW <= 16 ? 3 : 2);  // per SM
  static constexpr int kFixed = NWG * (kQBytes + kPBytes);
  // 227 KB a block, 228 KB an SM of which each block takes 1 KB and its
  // static variables; 1 KB to align.
  static constexpr int kBudget = (kCtas == 1 ? 227 : (228 - kCtas) / kCtas) * 1024 - 4096 - 1024;
  static constexpr int kSlots = (kBudget - kFixed) / kSlotBytes < 12 ? (kBudget - kFixed) / kSlotBytes : 12;
  static constexpr int kSmem = kSlots * kSlotBytes + kFixed + 1024;
  static_assert(kTmemUsed <= 512 && kTmemCols * kCtas <= 512, "TMEM of the resident blocks");
  static_assert(kSlots >= 4, "a K and a V tile in use and two on their way");
  static_assert(RW == 8 || RW == 16 || RW == 32, "rows of a warpgroup");
  static_assert(kN <= 128 && kSlotBytes % 1024 == 0 && kPBytes % 1024 == 0, "tile alignment");
};

struct Args {
  kv::CacheView c;
  const char* q;
  char* o;
  float* lse;
  long long q_sb, q_sh, q_ss, o_sb, o_sh, o_ss;
  int heads, group, seqlen_q;
  int prefix_mode;   // items are the shared prefix's (rows of all sequences)
  int key0;          // first key of these items
  int key_base;      // key0 rounded down to where a TMA box may start
  int prefix_len;
  int row_tiles;     // tiles of query rows per (sequence, K/V head)
  int box;           // keys of a TMA box: min(page_size, 128)
  int page_shift;    // log2(page_size), or -1
  int own_rows;      // results go to o (1), or to full_* and item (0)
  int early;         // this launch may overlap the one before it
  float scale_log2;
  long long timeout;
  float* part_o;     // [2 G][kRows][D] unnormalised sums of a block's first / last item
  float2* part_ml;   // [2 G][kRows]
  int4* seg;         // [G] the item that block c begins and another ends (own_rows)
  int4* item;        // [items] where each item's result is (!own_rows)
  float* full_o;     // [batch][heads][seqlen_q][D] unnormalised (!own_rows)
  float2* full_ml;
};

// ------------------------------------------------------------------ registers
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t* r) {
  if constexpr (N == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
    if constexpr (N > 16) tmem_ld<N - 16>(addr + 16, r + 16);
  }
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(
                   addr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
               "r"(r[7])
               : "memory");
}
// Uses of registers that a tcgen05.ld filled stay behind its wait.
template <int N>
__device__ __forceinline__ void wait_ld(uint32_t* r) {
  ptx::tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i])::"memory");
}

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint16_t e4m3x2_of_h2(uint32_t h) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(h));
  return r;
}
// 16 (x - t) in halves: both steps are exact (t has x's leading bits).
__device__ __forceinline__ uint32_t rest(uint32_t x, uint16_t t) {
  const uint32_t tb = ptx::cvt_e4m3x2_to_f16x2(t);
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&x),
                            *reinterpret_cast<const __half2*>(&tb));
  const __half2 s = __hmul2(d, __float2half2_rn(kTerm));
  return *reinterpret_cast<const uint32_t*>(&s);
}
// Terms of 8 values given as four half pairs: out[term] holds 8 bytes.
template <int NT>
__device__ __forceinline__ void terms8(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3,
                                       uint2 (&out)[NT]) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const uint16_t a = e4m3x2_of_h2(x0), b = e4m3x2_of_h2(x1), c = e4m3x2_of_h2(x2),
                   d = e4m3x2_of_h2(x3);
    out[t] = make_uint2((uint32_t)a | ((uint32_t)b << 16), (uint32_t)c | ((uint32_t)d << 16));
    if (t + 1 < NT) {
      x0 = rest(x0, a);
      x1 = rest(x1, b);
      x2 = rest(x2, c);
      x3 = rest(x3, d);
    }
  }
}
// Byte offset of column byte `col` of row `row` in a tile of rows of kPitch
// bytes under the 64 B or 128 B swizzle.
template <int kPitch>
__device__ __forceinline__ uint32_t swz(int row, int col) {
  const int chunk = col >> 4;
  const int x = kPitch == 128 ? (row & 7) : ((row >> 1) & 3);
  return (uint32_t)(row * kPitch + ((chunk ^ x) << 4) + (col & 15));
}

// Instruction descriptor of O^T += V^T P^T: both operands MN-major.
__host__ __device__ constexpr uint32_t idesc_tt(int m, int n) {
  return ptx::idesc_e4m3_f32(m, n, true) | (1u << 15);
}
// V^T as operand A: 128 rows of M out of tiles whose rows (keys) hold D bytes.
// D = 64 has half the rows: with a leading offset of zero rows 64..127 repeat
// rows 0..63.
template <int D>
__device__ __forceinline__ uint64_t desc_v(uint32_t addr) {
  uint64_t d = ptx::smem_desc_mnmajor(addr, D);
  if (D == 64) d &= ~(0x3FFFull << 16);
  return d;
}

// -------------------------------------------------------------------- waiting
// Every wait is bounded. One that gave up sets the block's abort flag, which
// ends all others; each role then leaves its loop.
struct Waiter {
  volatile int* abort;
  int* status;
  long long limit;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!ptx::mbar_try_wait_sleep(bar, parity, kWaitHintNs)) {
      if (*abort) return false;
      if (clock64() - t0 > limit) {
        *abort = 1;
        if (status) atomicOr(status, FA8_DEVERR_TIMEOUT);
        return false;
      }
    }
    return true;
  }
  // For a whole warp: one answer for all its lanes.
  __device__ __forceinline__ bool warp(uint64_t* bar, uint32_t parity) const {
    return __all_sync(0xffffffffu, (*this)(bar, parity));
  }
};
__device__ __forceinline__ void wait_quietly(uint64_t* bar, uint32_t parity, long long limit) {
  const long long t0 = clock64();
  while (!ptx::mbar_try_wait(bar, parity) && clock64() - t0 < limit) {
  }
}

// ----------------------------------------------------------------------- work
__device__ __forceinline__ int seq_len(const Args& a, int b) {
  if (a.prefix_mode) return a.prefix_len;
  const int len = __ldg(a.c.seqlens + b);
  return len < 0 || len > a.c.max_len ? -1 : len;
}
__device__ __forceinline__ int tiles_of(const Args& a, int len) {
  return len > a.key0 ? (len - a.key_base + kTileKeys - 1) / kTileKeys : 0;
}

// A run of key tiles t0..t1-1 of one item (sequence b, K/V head, row tile).
struct Seg {
  int b, hk, rt, t0, t1, nt, len;
  long long unit;  // number of tile t0 among all
};

// Walks a block's share of the tiles; every role of the block walks the same.
struct Walk {
  int b, hk, rt, t, nt, len;
  long long unit, left;
  __device__ __forceinline__ void enter(const Args& a) {
    len = seq_len(a, b);
    nt = tiles_of(a, len);
  }
  __device__ __forceinline__ void begin(const Args& a, int b0, long long off, long long unit0,
                                        long long units) {
    b = b0;
    unit = unit0;
    left = units;
    enter(a);
    const long long j = off / nt;
    t = (int)(off - j * nt);
    hk = (int)(j / a.row_tiles);
    rt = (int)(j - (long long)hk * a.row_tiles);
  }
  __device__ __forceinline__ bool next(const Args& a, Seg& s) {
    if (left == 0) return false;
    while (nt == 0) {
      ++b;
      enter(a);
    }
    s.b = b;
    s.hk = hk;
    s.rt = rt;
    s.t0 = t;
    s.nt = nt;
    s.len = len;
    s.t1 = (int)min((long long)nt, t + left);
    s.unit = unit;
    const int n = s.t1 - s.t0;
    left -= n;
    unit += n;
    t = s.t1;
    if (t == nt) {
      t = 0;
      if (++rt == a.row_tiles) {
        rt = 0;
        if (++hk == a.c.heads_kv) {
          hk = 0;
          ++b;
          if (left > 0) enter(a);
        }
      }
    }
    return true;
  }
};

__device__ __forceinline__ int page_of(const Args& a, int key) {
  return a.page_shift >= 0 ? key >> a.page_shift : key / a.c.page_size;
}

template <class C>
struct __align__(16) Shared {
  uint64_t kv_full[C::kSlots];
  uint64_t kv_empty[C::kSlots];
  uint64_t q_full[C::NWG];
  uint64_t s_full[C::NWG];   // S^T in TMEM
  uint64_t s_free[C::NWG];   // read by the four warps
  uint64_t p_full[C::NWG];   // P^T in shared memory (and O^T rescaled)
  uint64_t o_done[C::NWG];   // O^T += V^T P^T complete
  uint64_t meet[C::NWG];     // the four warps of a warpgroup
  uint64_t drain;
  uint32_t tmem;
  int abort;
  int b0;
  long long off0;
  long long warp_units[16];
  struct Group {
    float mul[C::RW];        // scale * log2(e) * the power of two of the row of Q
    float inv[C::RW];
    float sum[4][C::RW];
    float top[2][4][C::RW];  // warps' maxima of a tile, two tiles in turn
    long long o_off[C::RW];  // element offset of the row in o; -1: none
    int row_id[C::RW];       // (b * heads + h) * seqlen_q + i
    int lim[C::RW];          // keys that the row sees
  } g[C::NWG];
};

template <class C, bool kBf16>
__global__ void __launch_bounds__(C::kThreads, C::kCtas)
    decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const Args a) {
  constexpr int D = C::D, NT = C::NT, RW = C::RW, NS = C::kSlots;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared<C> sh;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int G = gridDim.x, cta = blockIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ------------------------------------------------- this block's share
  const int nseq = a.prefix_mode ? 1 : a.c.batch;
  const int chunk = (nseq + C::kThreads - 1) / C::kThreads;
  const int s0 = min(nseq, (int)threadIdx.x * chunk), s1 = min(nseq, s0 + chunk);
  const long long per = (long long)a.c.heads_kv * a.row_tiles;
  long long mine = 0;
  for (int b = s0; b < s1; ++b) {
    const int len = seq_len(a, b);
    if (len < 0 && cta == 0 && a.c.status) atomicOr(a.c.status, FA8_DEVERR_VARLEN_RANGE);
    mine += per * tiles_of(a, len);
  }
  long long upto = mine;  // inclusive scan
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sh.warp_units[warp] = upto;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      ptx::mbar_init(&sh.kv_full[s], 1);
      ptx::mbar_init(&sh.kv_empty[s], 1);
    }
    for (int w = 0; w < C::NWG; ++w) {
      ptx::mbar_init(&sh.q_full[w], 4);
      ptx::mbar_init(&sh.s_full[w], 1);
      ptx::mbar_init(&sh.s_free[w], 4);
      ptx::mbar_init(&sh.p_full[w], 4);
      ptx::mbar_init(&sh.o_done[w], 1);
      ptx::mbar_init(&sh.meet[w], 4);
    }
    ptx::mbar_init(&sh.drain, 1);
    sh.abort = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < C::kThreads / 32; ++w) {
    const long long v = sh.warp_units[w];
    if (w < warp) upto += v;
    total += v;
  }
  const long long shares = min((long long)G, total);  // blocks with work: a tile at least
  const long long u0 = cta < shares ? total * cta / shares : 0;
  const long long u1 = cta < shares ? total * (cta + 1) / shares : 0;
  if (u0 < u1 && u0 >= upto - mine && u0 < upto) {
    long long at = upto - mine;
    int b = s0;
    while (true) {
      const long long n = per * tiles_of(a, seq_len(a, b));
      if (u0 < at + n) break;
      at += n;
      ++b;
    }
    sh.b0 = b;
    sh.off0 = u0 - at;
  }

  // Sequences without a key among these items have no tile and no block of
  // their own: their rows (items) are filled in by block b mod G.
  if (!a.prefix_mode) {
    for (int b = cta; b < a.c.batch; b += G) {
      const int len = seq_len(a, b);
      if (len < 0 || tiles_of(a, len) > 0) continue;
      if (a.own_rows) {
        const int n = a.heads * a.seqlen_q;
        for (int j = threadIdx.x; j < n * (D / 8); j += C::kThreads) {
          const int row = j / (D / 8), h = row / a.seqlen_q, i = row - h * a.seqlen_q;
          reinterpret_cast<uint4*>(a.o + 2 * (b * a.o_sb + h * a.o_sh + i * a.o_ss))[j % (D / 8)] =
              make_uint4(0, 0, 0, 0);
          if (a.lse && j % (D / 8) == 0) a.lse[(long long)b * n + row] = -INFINITY;
        }
      } else {
        for (int j = threadIdx.x; j < per; j += C::kThreads)
          a.item[b * per + j] = make_int4(0, 0, 0, kItemEmpty);
      }
    }
  }
  if (a.own_rows && threadIdx.x == 0) a.seg[cta] = make_int4(-1, 0, 0, 0);
  if (u0 == u1) {
    if (a.early) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  // Ring of K and V tiles | P of each warpgroup | Q of each warpgroup.
  uint8_t* const p_tiles = smem + NS * C::kSlotBytes;
  uint8_t* const q_tiles = p_tiles + C::NWG * C::kPBytes;
  if (warp == C::kMmaWarp) {
    ptx::tmem_alloc(&sh.tmem, C::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const Waiter wait{&sh.abort, a.c.status, a.timeout};
  Walk walk;
  walk.begin(a, sh.b0, sh.off0, u0, u1 - u0);
  Seg s;

  if (warp == C::kLoadWarp) {
    // ------------------------------------------------------------ TMA producer
    // Lane l brings piece l (box keys of one page) of a K and of a V tile.
    // Ring item 2n is K of the block's tile n, 2n + 1 its V.
    const int pieces = kTileKeys / a.box;
    const uint64_t policy = a.row_tiles > 1 ? ptx::policy_evict_last() : ptx::policy_evict_first();
    if (lane == 0) {
      ptx::tma_prefetch_desc(&tm_k);
      ptx::tma_prefetch_desc(&tm_v);
    }
    int n = 0, issued = 0;
    bool ok = true;
    while (ok && walk.next(a, s)) {
      const int* table = a.c.table + (a.prefix_mode ? 0 : s.b) * a.c.table_stride;
      auto entry = [&](int t) {
        const int key = a.key_base + t * kTileKeys + lane * a.box;
        return lane < pieces && key < s.len ? __ldg(table + page_of(a, key)) : 0;
      };
      int page = entry(s.t0);
      for (int t = s.t0; t < s.t1; ++t, ++n) {
        const int next = t + 1 < s.t1 ? entry(t + 1) : 0;
        const int key = a.key_base + t * kTileKeys + lane * a.box;
        const bool have = lane < pieces && key < s.len;
        // A page outside the cache: coordinates that read as zeros.
        const int coord = page < 0 || page >= a.c.num_pages ? 0x7fffffff : page;
        const int slot = key - page_of(a, key) * a.c.page_size;
        const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, have)) * a.box * D;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int i = 2 * n + v, st = i % NS;
          if (lane == 0) {
            if (i >= NS) ok = wait(&sh.kv_empty[st], ((i / NS) - 1) & 1);
            if (ok) ptx::mbar_arrive_expect_tx(&sh.kv_full[st], bytes);
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          if (have)
            ptx::tma_load_4d(smem + st * C::kSlotBytes + lane * a.box * D, v ? &tm_v : &tm_k,
                             &sh.kv_full[st], 0, slot, s.hk, coord, policy);
          issued = i + 1;
        }
        if (!ok) break;
        page = next;
      }
    }
    if (!ok && lane == 0) {
      // Copies in flight land before the block ends.
      for (int i = max(0, issued - NS); i < issued; ++i)
        wait_quietly(&sh.kv_full[i % NS], (i / NS) & 1, a.timeout);
    }
  } else if (warp == C::kMmaWarp) {
    if (lane == 0) {
      // ------------------------------------------------------------ MMA issuer
      const uint32_t ring = ptx::smem_u32(smem), pb = ptx::smem_u32(p_tiles),
                     qb = ptx::smem_u32(q_tiles);
      constexpr uint32_t idesc_s = ptx::idesc_e4m3_f32(128, C::kN);
      constexpr uint32_t idesc_o = idesc_tt(128, C::kN);
      int n = 0, nseg = 0;
      bool ok = true;
      auto scores = [&](bool first) {  // S^T of tile n; `first` of its item
        const int i = 2 * n, st = i % NS;
        ok = wait(&sh.kv_full[st], (i / NS) & 1);
#pragma unroll
        for (int w = 0; w < C::NWG; ++w) {
          if (first) ok = ok && wait(&sh.q_full[w], nseg & 1);
          if (n > 0) ok = ok && wait(&sh.s_free[w], (n - 1) & 1);
          if (!ok) return;
          ptx::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 32; ++kk)
            ptx::umma_f8(tmem + w * 2 * C::kN,
                         ptx::smem_desc_kmajor(ring + st * C::kSlotBytes + kk * 32, D),
                         ptx::smem_desc_kmajor(qb + w * C::kQBytes + kk * 32, D), idesc_s,
                         kk > 0 ? 1u : 0u);
          ptx::umma_commit(&sh.s_full[w]);
        }
        ptx::umma_commit(&sh.kv_empty[st]);
      };
      auto values = [&](int m, bool first) {  // O^T += V^T P^T of tile m
        const int i = 2 * m + 1, st = i % NS;
        ok = wait(&sh.kv_full[st], (i / NS) & 1);
#pragma unroll
        for (int w = 0; w < C::NWG; ++w) {
          ok = ok && wait(&sh.p_full[w], m & 1);
          if (!ok) return;
          ptx::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < kTileKeys / 32; ++kk)
            ptx::umma_f8(tmem + w * 2 * C::kN + C::kN,
                         desc_v<D>(ring + st * C::kSlotBytes + kk * 32 * D),
                         ptx::smem_desc_mnmajor(pb + w * C::kPBytes + kk * 32 * C::kPitch, C::kPitch),
                         idesc_o, first && kk == 0 ? 0u : 1u);
          ptx::umma_commit(&sh.o_done[w]);
        }
        ptx::umma_commit(&sh.kv_empty[st]);
      };
      // The scores of the next tile are issued before this tile's values, so
      // that they are ready when the softmax of this one is done. The next
      // item's Q is written only after this item's last values.
      while (ok && walk.next(a, s)) {
        const int count = s.t1 - s.t0;
        scores(true);
        for (int j = 0; ok && j < count; ++j) {
          ++n;
          if (j + 1 < count) scores(false);
          if (ok) values(n - 1, j == 0);
        }
        ++nseg;
      }
      ptx::umma_commit(&sh.drain);
      wait_quietly(&sh.drain, 0, a.timeout);
    }
  } else {
    // --------------------------------------------------------------- softmax
    const int w = warp / 4, wq = warp % 4, tid = threadIdx.x % 128;
    auto& g = sh.g[w];
    // The warpgroup's own barrier, bounded like every other wait.
    uint32_t met = 0;
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sh.meet[w]);
      return wait.warp(&sh.meet[w], met++ & 1);
    };
    uint8_t* const p_tile = p_tiles + w * C::kPBytes;
    uint8_t* const q_tile = q_tiles + w * C::kQBytes;
    const uint32_t col_s = tmem + w * 2 * C::kN + ((uint32_t)(wq * 32) << 16), col_o = col_s + C::kN;
    int n = 0, nseg = 0;
    bool ok = true;
    while (ok && walk.next(a, s)) {
      ok = meet();  // the item before is done with g
      if (!ok) break;
      // ------------------------------------------------ rows and Q of the item
      const int rows_seq = a.seqlen_q * a.group;
      const int rows = rows_seq * (a.prefix_mode ? a.c.batch : 1);
      const int row0 = s.rt * C::kRows + w * RW;
      if (tid < RW) {
        const int j = row0 + tid;
        int lim = s.len, id = -1;
        long long off = -1;
        if (j < rows) {
          const int b = a.prefix_mode ? j / rows_seq : s.b;
          const int r = a.prefix_mode ? j - b * rows_seq : j;
          const int i = r / a.group, h = s.hk * a.group + r - i * a.group;
          int len = s.len;
          if (a.prefix_mode) {
            len = __ldg(a.c.seqlens + b);
            if (len > a.c.max_len) len = 0;  // refused: its rows are not joined
          }
          lim = max(0, min(s.len, len - a.seqlen_q + i + 1));
          id = (b * a.heads + h) * a.seqlen_q + i;
          off = b * a.o_sb + h * a.o_sh + i * a.o_ss;
        }
        g.lim[tid] = lim;
        g.row_id[tid] = id;
        g.o_off[tid] = off;
      }
      constexpr int kLanes = D / 8;  // lanes of a row of Q
#pragma unroll
      for (int pass = 0; pass < (RW * kLanes + 127) / 128; ++pass) {
        const int r = (pass * 128 + tid) / kLanes, cl = tid % kLanes;
        const int j = row0 + r;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < RW && j < rows) {
          const int b = a.prefix_mode ? j / rows_seq : s.b;
          const int rr = a.prefix_mode ? j - b * rows_seq : j;
          const int i = rr / a.group, h = s.hk * a.group + rr - i * a.group;
          x = __ldg(reinterpret_cast<const uint4*>(
                        a.q + 2 * (b * a.q_sb + h * a.q_sh + i * a.q_ss)) + cl);
        }
        uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                              __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
        m = max(m & 0xffffu, m >> 16);
#pragma unroll
        for (int o = kLanes / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const bool fine = m < (kBf16 ? 0x7f80u : 0x7c00u);
        const uint32_t bits =
            kBf16 ? m << 16
                  : __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
        // 2^(7 - e) with 2^e <= max < 2^(e + 1); rows below 2^-100 are as good as zero.
        const int e = m == 0 ? 7 : max((int)(bits >> 23) - 127, -100);
        const float f = fine ? __uint_as_float((uint32_t)(127 + 7 - e) << 23) : 0.f;
        uint32_t hx[4];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const uint32_t word = q4 == 0 ? x.x : q4 == 1 ? x.y : q4 == 2 ? x.z : x.w;
          float2 v;
          if (kBf16)
            v = make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
          else
            v = __half22float2(*reinterpret_cast<const __half2*>(&word));
          hx[q4] = fine ? h2(v.x * f, v.y * f) : 0u;
        }
        uint2 t8[NT];
        terms8<NT>(hx[0], hx[1], hx[2], hx[3], t8);
        if (r < RW) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
            *reinterpret_cast<uint2*>(q_tile + swz<D>(t * RW + r, cl * 8)) = t8[t];
          if (cl == 0)
            g.mul[r] = fine ? a.scale_log2 * __uint_as_float((uint32_t)(127 - 7 + e) << 23)
                            : __int_as_float(0x7fc00000);
        }
      }
      ptx::fence_proxy_async_smem();
      ok = meet();  // mul, lim and row_id are there for all
      if (!ok) break;
      if (lane == 0) ptx::mbar_arrive(&sh.q_full[w]);
      int all_see = s.len;  // keys that every row sees
#pragma unroll
      for (int r = 0; r < RW; ++r) all_see = min(all_see, g.lim[r]);

      const int* table = a.c.table + (a.prefix_mode ? 0 : s.b) * a.c.table_stride;
      const uint8_t* ke = a.c.k_exp + s.hk * a.c.ke_sh;
      const uint8_t* ve = a.c.v_exp + s.hk * a.c.ve_sh;
      // Page of this thread's key in tile t, and the key's exponent bytes
      // (K in the low half): both asked for one tile before they are needed.
      auto page_at = [&](int t) {
        const int key = a.key_base + t * kTileKeys + tid;
        return key < s.len && t < s.t1 ? __ldg(table + page_of(a, key)) : 0;
      };
      auto bytes_at = [&](int t, int page) -> uint32_t {
        const int key = a.key_base + t * kTileKeys + tid;
        if (key >= s.len || key < a.key0 || t >= s.t1) return 127u | (127u << 16);
        if (page < 0 || page >= a.c.num_pages) {
          if (a.c.status) atomicOr(a.c.status, FA8_DEVERR_PAGE_RANGE);
          return 255u | (255u << 16);
        }
        const int slot = key - page_of(a, key) * a.c.page_size;
        return (uint32_t)__ldg(ke + page * a.c.ke_sp + slot) |
               ((uint32_t)__ldg(ve + page * a.c.ve_sp + slot) << 16);
      };
      uint32_t eb_next = bytes_at(s.t0, page_at(s.t0));
      int page_next = page_at(s.t0 + 1);

      float m[RW], l[RW];
      float m_lane = -INFINITY;  // running maximum of row `lane`
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        m[r] = 0.f;
        l[r] = 0.f;
      }
      for (int t = s.t0; t < s.t1; ++t, ++n) {
        const uint32_t eb = eb_next;
        eb_next = bytes_at(t + 1, page_next);
        page_next = page_at(t + 2);
        const int key = a.key_base + t * kTileKeys + tid;
        const float kf = kv::exp_factor((int)(eb & 0xffffu));
        const int vb = (int)(eb >> 16);
        const float vexp = vb == kv::kExpNan ? 0.f : (float)(vb - kv::kExpBias);
        const float vf = kv::exp_factor(vb) * kPScale;
        // Every key of the tile seen by every row?
        const int first_key = a.key_base + t * kTileKeys;
        const bool plain = first_key >= a.key0 && first_key + kTileKeys <= all_see;

        ok = wait.warp(&sh.s_full[w], n & 1);
        if (!ok) break;
        ptx::tc_fence_after();
        float x[RW];
        {
          uint32_t raw[NT * RW];
#pragma unroll
          for (int q = 0; q < NT; ++q) tmem_ld<RW>(col_s + q * RW, raw + q * RW);
          wait_ld<NT * RW>(raw);
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&sh.s_free[w]);
#pragma unroll
          for (int r = 0; r < RW; ++r) {
            float v = __uint_as_float(raw[(NT - 1) * RW + r]);
#pragma unroll
            for (int q = NT - 2; q >= 0; --q)
              v = fmaf(v, 1.f / kTerm, __uint_as_float(raw[q * RW + r]));
            x[r] = v * (kf * g.mul[r]);
          }
        }
        if (!plain) {
#pragma unroll
          for (int r = 0; r < RW; ++r)
            if (key < a.key0 || key >= g.lim[r]) x[r] = -INFINITY;
        }
        // Largest s + e of each row over the tile, against the running one.
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          const float v = warp_max(x[r] + vexp);
          if (lane == r) top = v;
        }
        if (lane < RW) g.top[n & 1][wq][lane] = top;
        ok = meet();
        if (!ok) break;
        float f_lane = 1.f;
        bool up = false;
        if (lane < RW) {
          const float v = fmaxf(fmaxf(g.top[n & 1][0][lane], g.top[n & 1][1][lane]),
                                fmaxf(g.top[n & 1][2][lane], g.top[n & 1][3][lane]));
          up = v > m_lane + kRise;
          if (up) {
            f_lane = m_lane == -INFINITY ? 0.f : ptx::ex2(m_lane - v);
            m_lane = v;
          }
        }
        // The values of the tile before are complete: P may be overwritten and
        // O rescaled.
        const bool any_up = __any_sync(0xffffffffu, up);
        if (n > 0) {
          ok = wait.warp(&sh.o_done[w], (n - 1) & 1);
          if (!ok) break;
        }
        if (any_up) {
          if (t > s.t0) {
            ptx::tc_fence_after();
#pragma unroll
            for (int q = 0; q < NT; ++q) {
#pragma unroll
              for (int c = 0; c < RW; c += 8) {
                uint32_t o8[8];
                tmem_ld<8>(col_o + q * RW + c, o8);
                wait_ld<8>(o8);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  o8[k] = __float_as_uint(__uint_as_float(o8[k]) *
                                          __shfl_sync(0xffffffffu, f_lane, c + k));
                tmem_st8(col_o + q * RW + c, o8);
              }
            }
            ptx::tmem_wait_st();
          }
          const float use = m_lane == -INFINITY ? 0.f : m_lane;
#pragma unroll
          for (int r = 0; r < RW; ++r) {
            l[r] *= __shfl_sync(0xffffffffu, f_lane, r);
            m[r] = __shfl_sync(0xffffffffu, use, r);
          }
        }
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          const float p = ptx::ex2(x[r] - m[r]);
          l[r] += p;
          // A masked key's factor may be anything: its product is not formed.
          x[r] = !plain && x[r] == -INFINITY ? 0.f : p * vf;
        }
        // The key's row of P: the terms side by side.
#pragma unroll
        for (int c = 0; c < RW; c += 8) {
          uint2 t8[NT];
          terms8<NT>(h2(x[c], x[c + 1]), h2(x[c + 2], x[c + 3]), h2(x[c + 4], x[c + 5]),
                     h2(x[c + 6], x[c + 7]), t8);
#pragma unroll
          for (int q = 0; q < NT; ++q)
            *reinterpret_cast<uint2*>(p_tile + swz<C::kPitch>(tid, q * RW + c)) = t8[q];
        }
        // Rows of V that are not this item's keys (the end of a page, a page
        // not brought in) may hold anything, NaN codes among them: zeros.
        if (w == 0 && (first_key < a.key0 || first_key + kTileKeys > s.len)) {
          const int st = (2 * n + 1) % NS;
          ok = wait.warp(&sh.kv_full[st], ((2 * n + 1) / NS) & 1);
          if (!ok) break;
          if (key < a.key0 || key >= s.len) {
            uint4* row = reinterpret_cast<uint4*>(smem + st * C::kSlotBytes + tid * D);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) row[c] = make_uint4(0, 0, 0, 0);
          }
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sh.p_full[w]);
      }
      if (!ok) break;

      // ------------------------------------------------------ the item's result
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        float v = l[r];
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == r) g.sum[wq][r] = v;
      }
      ok = wait.warp(&sh.o_done[w], (n - 1) & 1);
      if (!ok) break;
      ptx::tc_fence_after();
      ok = meet();
      if (!ok) break;
      const bool begins = s.t0 == 0, whole = begins && s.t1 == s.nt;
      const int part = 2 * cta + (nseg > 0 ? 1 : 0);
      if (tid < RW) {
        const float sum = (g.sum[0][tid] + g.sum[1][tid]) + (g.sum[2][tid] + g.sum[3][tid]);
        // Row `tid` is row `lane` of warp 0, whose lanes hold the maxima.
        const float top = sum == 0.f ? -INFINITY : (m_lane == -INFINITY ? 0.f : m_lane);
        const int id = g.row_id[tid];
        if (!whole) {
          a.part_ml[(long long)part * C::kRows + w * RW + tid] = make_float2(top, sum);
        } else if (!a.own_rows) {
          if (id >= 0) a.full_ml[id] = make_float2(top, sum);
        } else {
          g.inv[tid] = sum == 0.f ? 0.f : 1.f / (kPScale * sum);
          if (id >= 0 && a.lse)
            a.lse[id] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
        }
      }
      if (w == 0 && tid == 0) {
        // Block that holds the item's last tile: the last c with U c / G < unit + 1.
        auto last_block = [&](long long unit) {
          return (int)(((unit + 1) * shares - 1) / total);
        };
        if (a.own_rows) {
          if (begins && !whole)
            a.seg[cta] = make_int4(last_block(s.unit + s.nt - 1), s.b,
                                   s.hk * a.row_tiles + s.rt, part);
        } else if (begins) {
          a.item[(long long)s.b * per + s.hk * a.row_tiles + s.rt] =
              make_int4(cta, whole ? cta : last_block(s.unit + s.nt - 1), part,
                        whole ? kItemFull : kItemParts);
        }
      }
      ok = meet();
      if (!ok) break;
      // O^T: a thread has one d of every row; with D = 64 the upper half of the
      // lanes repeats the lower and takes the odd rows.
      const int d = tid % D;
      const bool own_half = D == 128;
#pragma unroll
      for (int c = 0; c < RW; c += 8) {
        uint32_t raw[NT * 8];
#pragma unroll
        for (int q = 0; q < NT; ++q) tmem_ld<8>(col_o + q * RW + c, raw + q * 8);
        wait_ld<NT * 8>(raw);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float v = __uint_as_float(raw[(NT - 1) * 8 + k]);
#pragma unroll
          for (int q = NT - 2; q >= 0; --q)
            v = fmaf(v, 1.f / kTerm, __uint_as_float(raw[q * 8 + k]));
          const int r = c + k;
          const int id = g.row_id[r];
          if (id < 0 || !(own_half || (r & 1) == tid / 64)) continue;
          if (!whole) {
            a.part_o[((long long)part * C::kRows + w * RW + r) * D + d] = v;
          } else if (!a.own_rows) {
            a.full_o[(long long)id * D + d] = v;
          } else {
            const float y = v * g.inv[r];
            if (kBf16)
              reinterpret_cast<__nv_bfloat16*>(a.o)[g.o_off[r] + d] = __float2bfloat16(y);
            else
              reinterpret_cast<__half*>(a.o)[g.o_off[r] + d] = __float2half(y);
          }
        }
      }
      ptx::tc_fence_before();
      ++nseg;
    }
  }

  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, C::kTmemCols);
  }
  // A launch that overlaps the one before it ends after it: whoever waits for
  // this one has both.
  if (a.early) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// --------------------------------------------------------------------- joining
// Sum of parts of one row, spread over a warp: lane holds D / 32 values.
template <int D>
struct RowSum {
  static constexpr int V = D / 32;
  float m = -INFINITY, l = 0.f, o[V];
  __device__ __forceinline__ RowSum() {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.f;
  }
  __device__ __forceinline__ static void load(const float* p, float (&x)[V]) {
    if constexpr (V == 4) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p));
      x[0] = v.x;
      x[1] = v.y;
      x[2] = v.z;
      x[3] = v.w;
    } else {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(p));
      x[0] = v.x;
      x[1] = v.y;
    }
  }
  // Parts i < n; at(i) gives the row's index in the part arrays.
  template <class At>
  __device__ __forceinline__ void add(const float* po, const float2* pml, int n, At at) {
    const int lane = threadIdx.x % 32;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int here = min(32, n - i0);
      float2 ml = make_float2(-INFINITY, 0.f);
      if (lane < here) ml = __ldcg(pml + at(i0 + lane));
      const float top = fmaxf(m, warp_max(ml.x));
      const float use = top == -INFINITY ? 0.f : top;
      const float keep = ptx::ex2(m - use), w = ptx::ex2(ml.x - use);
      float sum = w * ml.y;
#pragma unroll
      for (int k = 16; k; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
      l = l * keep + sum;
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] *= keep;
      m = top;
#pragma unroll 4
      for (int i = 0; i < here; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        float x[V];
        load(po + at(i0 + i) * D + lane * V, x);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf(wi, x[e], o[e]);
      }
    }
  }
  template <bool kBf16>
  __device__ __forceinline__ void store(const Args& a, int b, int h, int i) const {
    const int lane = threadIdx.x % 32;
    const float inv = l == 0.f ? 0.f : 1.f / (kPScale * l);
    uint32_t w[V / 2];
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      if (kBf16) {
        const __nv_bfloat162 y = __floats2bfloat162_rn(o[e] * inv, o[e + 1] * inv);
        w[e / 2] = *reinterpret_cast<const uint32_t*>(&y);
      } else {
        w[e / 2] = h2(o[e] * inv, o[e + 1] * inv);
      }
    }
    char* dst = a.o + 2 * (b * a.o_sb + h * a.o_sh + i * a.o_ss + lane * V);
    if constexpr (V == 4)
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(dst) = w[0];
    if (a.lse && lane == 0)
      a.lse[((long long)b * a.heads + h) * a.seqlen_q + i] =
          l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
};

// Joins the parts of the item that block `blockIdx.x` of the first kernel
// began and did not end; a warp per row.
template <int D, bool kBf16>
__global__ void __launch_bounds__(128) decode_join_kernel(const Args a, int tile_rows) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 s = __ldcg(a.seg + blockIdx.x);  // last block, sequence, head and row tile, part
  if (s.x < 0) return;
  const int hk = s.z / a.row_tiles, rt = s.z - hk * a.row_tiles;
  const int r = blockIdx.y * 4 + threadIdx.x / 32, j = rt * tile_rows + r;
  if (r >= tile_rows || j >= a.seqlen_q * a.group) return;
  const int c0 = blockIdx.x;
  RowSum<D> sum;
  sum.add(a.part_o, a.part_ml, s.x - c0 + 1, [&](int k) {
    return (long long)(k == 0 ? s.w : 2 * (c0 + k)) * tile_rows + r;
  });
  sum.template store<kBf16>(a, s.y, hk * a.group + j % a.group, j / a.group);
}

// The items of one of the two sets that the joining kernel reads.
struct Set {
  const int4* item;
  const float* full_o;
  const float2* full_ml;
  const float* part_o;
  const float2* part_ml;
  int row_tiles, tile_rows;
};

// Joins every row's prefix with what is behind it; a warp per row.
template <int D, bool kBf16>
__global__ void __launch_bounds__(128) prefix_join_kernel(const Args a, const Set pre, const Set own) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int id = blockIdx.x * 4 + threadIdx.x / 32;
  if (id >= a.c.batch * a.heads * a.seqlen_q) return;
  const int i = id % a.seqlen_q, bh = id / a.seqlen_q, h = bh % a.heads, b = bh / a.heads;
  const int len = __ldg(a.c.seqlens + b);
  if (len < 0 || len > a.c.max_len) return;
  const int hk = h / a.group, j = i * a.group + h % a.group;
  RowSum<D> sum;
  auto take = [&](const Set& s, int row, int seq) {
    const int4 it = __ldcg(s.item + ((long long)seq * a.c.heads_kv + hk) * s.row_tiles +
                           row / s.tile_rows);
    if (it.w == kItemFull) {
      sum.add(s.full_o, s.full_ml, 1, [&](int) { return (long long)id; });
    } else if (it.w == kItemParts) {
      sum.add(s.part_o, s.part_ml, it.y - it.x + 1, [&](int k) {
        return (long long)(k == 0 ? it.z : 2 * (it.x + k)) * s.tile_rows + row % s.tile_rows;
      });
    }
  };
  take(pre, b * a.seqlen_q * a.group + j, 0);
  take(own, j, b);
  sum.template store<kBf16>(a, b, h, i);
}

// ------------------------------------------------------------------------ host
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

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// Codes as {d, slots, heads, pages}, boxes of `box` slots, swizzled by rows.
int make_map(CUtensorMap* map, const fa8_kv_cache& c, const void* base, int64_t sp, int64_t sh,
             int64_t ss, int box, const void* dummy) {
  auto enc = encode_fn();
  if (!enc) return fa8_note_error(FA8_ERR_DRIVER, "cuTensorMapEncodeTiled entry point not found");
  // A cache without pages: nothing is read, but a map needs an address.
  if (c.num_pages == 0) base = dummy;
  cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.heads_kv,
                        (cuuint64_t)std::max<int64_t>(c.num_pages, 1)};
  cuuint64_t strides[3] = {(cuuint64_t)ss, (cuuint64_t)sh, (cuuint64_t)sp};
  cuuint32_t boxes[4] = {(cuuint32_t)c.head_dim, (cuuint32_t)box, 1, 1};
  cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult r =
      enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, boxes,
          ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
          c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    char msg[96];
    snprintf(msg, sizeof(msg), "fa8_decode: cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
    return fa8_note_error(FA8_ERR_ALIGNMENT, msg);
  }
  return FA8_OK;
}

// Row shape of a set of items: rows of a tile, its launch and its grid.
struct Shape {
  int rw, nwg;
  int tile_rows() const { return rw * nwg; }
};
Shape shape_for(int64_t rows) {
  if (rows <= 8) return {8, 1};
  if (rows <= 16) return {16, 1};
  if (rows <= 32) return {32, 1};
  return {32, 2};
}
int ctas_per_sm(int64_t d, const Shape& s) { return s.nwg > 1 ? 1 : (d == 64 && s.rw <= 16 ? 3 : 2); }

constexpr int kSmCount = 148;

// Workspace of one set of items.
struct Layout {
  Shape shape;
  int64_t row_tiles, items, grid;
  int64_t part_o, part_ml, seg, item, full_o, full_ml, end;  // byte offsets
};
int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

Layout layout_of(const fa8_decode_params* p, bool prefix_set, int64_t at) {
  Layout l;
  const int64_t D = p->cache.head_dim, B = p->cache.batch;
  const int64_t rows = p->seqlen_q * (p->heads / p->cache.heads_kv) * (prefix_set ? B : 1);
  l.shape = shape_for(rows);
  l.row_tiles = (rows + l.shape.tile_rows() - 1) / l.shape.tile_rows();
  l.items = p->cache.heads_kv * l.row_tiles * (prefix_set ? 1 : B);
  l.grid = (int64_t)kSmCount * ctas_per_sm(D, l.shape);
  const int64_t parts = 2 * l.grid * l.shape.tile_rows();
  const bool two = p->prefix_len > 0;
  const int64_t all = B * p->heads * p->seqlen_q;
  l.part_o = at;
  l.part_ml = l.part_o + up256(parts * D * 4);
  l.seg = l.part_ml + up256(parts * 8);
  l.item = l.seg + up256(l.grid * 16);
  l.full_o = l.item + (two ? up256(l.items * 16) : 0);
  l.full_ml = l.full_o + (two ? up256(all * D * 4) : 0);
  l.end = l.full_ml + (two ? up256(all * 8) : 0);
  return l;
}

template <class K, class... A>
cudaError_t launch_early(K kernel, dim3 grid, int threads, int smem, cudaStream_t stream, bool early,
                         const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = early ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e == cudaSuccess) fa8_note_launch();
  return e;
}

template <class C, bool kBf16>
int launch_set(const Args& a, const CUtensorMap& tk, const CUtensorMap& tv, int grid, int dev,
               cudaStream_t stream) {
  static std::once_flag flags[64];
  static cudaError_t errs[64];
  if (dev < 0 || dev >= 64) return fa8_note_error(FA8_ERR_INVALID_ARG, "device index out of range");
  auto kernel = decode_kernel<C, kBf16>;
  std::call_once(flags[dev], [&] {
    errs[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (errs[dev] != cudaSuccess) return fa8_note_cuda_error(errs[dev], "cudaFuncSetAttribute");
  const cudaError_t e = launch_early(kernel, dim3((unsigned)grid), C::kThreads, C::kSmem, stream,
                                     a.early != 0, tk, tv, a);
  return e == cudaSuccess ? FA8_OK : fa8_note_cuda_error(e, "decode kernel launch");
}

template <int D, bool kBf16>
int run_set(const fa8_decode_params* p, Args a, const Layout& l, char* ws, int dev,
            cudaStream_t stream) {
  constexpr int NT = kBf16 ? 2 : 3;
  const fa8_kv_cache& c = p->cache;
  a.row_tiles = (int)l.row_tiles;
  a.part_o = reinterpret_cast<float*>(ws + l.part_o);
  a.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
  a.seg = reinterpret_cast<int4*>(ws + l.seg);
  a.item = reinterpret_cast<int4*>(ws + l.item);
  a.full_o = reinterpret_cast<float*>(ws + l.full_o);
  a.full_ml = reinterpret_cast<float2*>(ws + l.full_ml);
  CUtensorMap tk, tv;
  int st = make_map(&tk, c, c.k, c.k_stride_p, c.k_stride_h, c.k_stride_s, a.box, ws);
  if (!st) st = make_map(&tv, c, c.v, c.v_stride_p, c.v_stride_h, c.v_stride_s, a.box, ws);
  if (st) return st;
  const int grid = (int)l.grid;
  if (l.shape.nwg == 2) return launch_set<Cfg<D, NT, 32, 2>, kBf16>(a, tk, tv, grid, dev, stream);
  if (l.shape.rw == 32) return launch_set<Cfg<D, NT, 32, 1>, kBf16>(a, tk, tv, grid, dev, stream);
  if (l.shape.rw == 16) return launch_set<Cfg<D, NT, 16, 1>, kBf16>(a, tk, tv, grid, dev, stream);
  return launch_set<Cfg<D, NT, 8, 1>, kBf16>(a, tk, tv, grid, dev, stream);
}

template <int D, bool kBf16>
int run(const fa8_decode_params* p, Args a, char* ws, int dev, cudaStream_t stream) {
  cudaError_t e;
  if (p->prefix_len == 0) {
    const Layout l = layout_of(p, false, 0);
    a.own_rows = 1;
    const int st = run_set<D, kBf16>(p, a, l, ws, dev, stream);
    if (st) return st;
    a.row_tiles = (int)l.row_tiles;
    a.part_o = reinterpret_cast<float*>(ws + l.part_o);
    a.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
    a.seg = reinterpret_cast<int4*>(ws + l.seg);
    const int rows = l.shape.tile_rows();
    e = launch_early(decode_join_kernel<D, kBf16>,
                     dim3((unsigned)l.grid, (unsigned)((std::min<int64_t>(
                                                rows, p->seqlen_q * a.group) + 3) / 4)),
                     128, 0, stream, true, a, rows);
  } else {
    const Layout l0 = layout_of(p, true, 0), l1 = layout_of(p, false, l0.end);
    Args b = a;
    b.prefix_mode = 1;
    int st = run_set<D, kBf16>(p, b, l0, ws, dev, stream);
    if (st) return st;
    b = a;
    b.key0 = a.prefix_len;
    b.key_base = a.prefix_len / a.box * a.box;
    b.early = 1;
    st = run_set<D, kBf16>(p, b, l1, ws, dev, stream);
    if (st) return st;
    auto set = [&](const Layout& l) {
      Set s;
      s.item = reinterpret_cast<const int4*>(ws + l.item);
      s.full_o = reinterpret_cast<const float*>(ws + l.full_o);
      s.full_ml = reinterpret_cast<const float2*>(ws + l.full_ml);
      s.part_o = reinterpret_cast<const float*>(ws + l.part_o);
      s.part_ml = reinterpret_cast<const float2*>(ws + l.part_ml);
      s.row_tiles = (int)l.row_tiles;
      s.tile_rows = l.shape.tile_rows();
      return s;
    };
    const int64_t rows = p->cache.batch * p->heads * p->seqlen_q;
    e = launch_early(prefix_join_kernel<D, kBf16>, dim3((unsigned)((rows + 3) / 4)), 128, 0, stream,
                     true, a, set(l0), set(l1));
  }
  return e == cudaSuccess ? FA8_OK : fa8_note_cuda_error(e, "decode join kernel launch");
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
  using namespace fa8::dec;
  if (!p || p->cache.batch < 0 || p->heads < 0 || p->seqlen_q < 0 || p->prefix_len < 0 ||
      (p->cache.head_dim != 64 && p->cache.head_dim != 128) || p->cache.heads_kv <= 0 ||
      p->heads % p->cache.heads_kv != 0) {
    fa8_note_error(FA8_ERR_INVALID_ARG, "fa8_decode_workspace_size: sizes that fa8_decode refuses");
    return -1;
  }
  if (p->cache.batch == 0 || p->heads == 0 || p->seqlen_q == 0) return 0;
  if (p->prefix_len == 0) return layout_of(p, false, 0).end;
  return layout_of(p, false, layout_of(p, true, 0).end).end;
}

int fa8_decode(const fa8_decode_params* p, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace fa8::dec;
  bool empty;
  int st = check(p, &empty);
  if (st || empty) return st;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
      workspace_bytes < fa8_decode_workspace_size(p))
    return fa8_note_error(FA8_ERR_INVALID_ARG,
                          "fa8_decode needs a 256-byte aligned workspace of "
                          "fa8_decode_workspace_size() bytes");
  st = fa8::kv::check_device();
  if (st) return st;
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return fa8_note_cuda_error(e, "cudaGetDevice");
  Args a = Args();
  a.c = fa8::kv::view_of(p->cache);
  a.q = static_cast<const char*>(p->q);
  a.o = static_cast<char*>(p->o);
  a.lse = p->lse;
  a.heads = (int)p->heads;
  a.group = (int)(p->heads / p->cache.heads_kv);
  a.seqlen_q = (int)p->seqlen_q;
  a.prefix_len = (int)p->prefix_len;
  const int page = (int)p->cache.page_size;
  a.box = std::min(page, kTileKeys);
  a.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (page == 1 << s) a.page_shift = s;
  a.q_sb = p->q_stride_b;
  a.q_sh = p->q_stride_h;
  a.q_ss = p->q_stride_s;
  a.o_sb = p->o_stride_b;
  a.o_sh = p->o_stride_h;
  a.o_ss = p->o_stride_s;
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  a.timeout = p->wait_timeout_cycles > 0 ? p->wait_timeout_cycles : kTimeout;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const bool bf16 = p->dtype == FA8_DT_BF16;
  if (p->cache.head_dim == 128)
    return bf16 ? run<128, true>(p, a, ws, dev, s) : run<128, false>(p, a, ws, dev, s);
  return bf16 ? run<64, true>(p, a, ws, dev, s) : run<64, false>(p, a, ws, dev, s);
}

}  // extern "C"
