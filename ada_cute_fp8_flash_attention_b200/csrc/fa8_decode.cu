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
// then holds one key: its two exponent bytes and its row of P^T.
//
// Rows to 8 bits. tcgen05 wants Q and P in e4m3 too. A value x is held as
// terms x = t0 + t1 / 16 + t2 / 256, t0 = rn(x), t1 = rn(16 (x - t0)), ...;
// e4m3 has 4 significant bits and a rounding is off by half a step, so two
// terms hold 8 bits and three hold 11 or more: what bf16 and fp16 have. The
// terms are columns of their own (N is 2 or 3 times the rows) and are added
// up in fp32 with their weights. Q is scaled by a power of two per row so that
// its largest magnitude is in [128, 256). The last term's least step is 2^-13
// (bf16) or 2^-17 (fp16) there: elements from 2^-13 or 2^-14 of the largest up
// are held exactly, smaller ones to 2^-21 or 2^-25 of it. P is rounded once to 11
// (fp16) or 8 (bf16) bits, as it would be for a 16-bit product.
//
// Softmax in base 2 with one running maximum per row, m = max(s + e), e the
// exponent of v_j over kRef, that of rows of unit normal values: then
// p = 2^(s - m) enters the sum, and what goes to the product is 8 * 2^e * p <= 8
// whatever the exponents are (times 2^5, the rise of a maximum that is let be:
// nothing is looked at row by row, exchanged or rescaled before one rises
// further). Half the least step of the last term, 2^-10 / 16 or 2^-10 / 256, is
// then 2^-17 (bf16) or 2^-21 (fp16) of the row's largest: the floor under small
// p. The sum is kept per thread, over its own keys, in fp32, and joined at the
// end of a row's keys.
//
// The largest p is as far from 1 as e is from 0: within 2^40 the sum has room
// and keeps its digits. Where a key's exponent is further away (rows of V below
// 1e-12 or above 1e12), or a row of zeros (whose exponent says nothing) has a
// score so high that it would set the maximum, the block computes its share once
// more in fp32 when it is done (share_again): values of any size beside each
// other are right, at a price that others do not pay. A reference of the item's
// own, its first tile's largest exponent, cost every call 2 to 3 % more.
//
// A block: one or more softmax warpgroups (8 or 16 rows each), a warp that
// brings tiles, a thread that issues products, two warps that prepare the next
// item's Q. The scores of tile n + 1 are issued before the values of tile n.
// Registers go from the helpers to the softmax (setmaxnreg). 8 and 16 rows
// have two blocks an SM (D = 64 and 8 rows three: its tile is half as large
// and is gone twice as fast), 32 rows two warpgroups, more rows four in one
// block, whose products are joint: an instruction costs the issuing thread
// some 100 clocks whatever its N.
//
// Work. Key tiles of 128 of all items (sequence, K/V head, tile of query rows)
// are numbered through, an item weighing a few tiles for itself, and every
// block takes an equal run of them, which it finds from the lengths on the
// device by a scan: any mixture of lengths shares the GPU evenly and nothing is
// read on the host. A block that holds all of an item's keys writes the result;
// else it writes its unnormalised sums, and a second kernel, launched early and
// waiting on the device for the first, joins them (always the same shares:
// results repeat bit by bit).
//
// The whole pages of a shared prefix are one more set of items, whose rows are
// those of the whole batch: one launch for it, one for what is behind it, one that
// joins both. A prefix of few tiles is left in each sequence's own items
// (prefix_apart).
//
// Measured on B200, inputs in turn: 64 sequences of up to 16384 keys, 32 heads on
// 8, bf16, 1.15 GB of cache: 177 us replayed from a graph, 6.5 TB/s, the copy rate
// measured beside it; 181 to 192 us called from Python one after another (over
// boxes; 185 where the graph took 177), 6.0 to 6.3 TB/s. One sequence of 131072
// keys, 32 heads on 4: 33 us replayed, 4.1 TB/s: some 5 us until the first product
// and as many from the last to the joined result are what a call costs that is this
// short. 64 sequences behind 16384 shared keys: 89 us; there the chain of a tile
// (scores, maximum test, exponentials, terms, values) in front of 64 rows bounds
// it, about 3000 clocks, of which the exponentials take 512.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "fa8_kv.cuh"
#include "sm100_ptx.cuh"

namespace fa8 {
namespace dec {

using kv::Divisor;

constexpr int kTileKeys = 128;
constexpr int kMostItemCost = 8;
constexpr int kAgainBar = 6;           // named barrier of share_again
constexpr int kMostWarps = 16;         // that prepare Q, or of the softmax
constexpr float kRise = 5.f;           // log2 of the rise of a maximum that is let be
constexpr int kPShift = 3;             // 8 p 2^e <= 2^(3 + kRise) < 448
constexpr int kRef = -7;               // exponents of V are taken over: that of unit normal rows
constexpr float kWide = 40.f;          // how far from it they may be
constexpr float kTerm = 16.f;          // weight of a term over the next
constexpr long long kTimeout = 4000000000LL;
constexpr int kWaitHintNs = 20000;

// Where an item's result is, for the kernel that joins the prefix with what is
// behind it.
enum { kItemEmpty = 0, kItemFull = 1, kItemParts = 2 };

// Blocks an SM holds: what four warpgroups leave of TMEM, else what registers
// and the ring do (D = 64 has half the tile, and needs more of them in flight).
constexpr int resident(int d, int rw, int nwg) {
  return nwg > 2 ? 1 : (d == 64 && rw == 8 ? 3 : 2);
}

// D: head dimension. NT: e4m3 terms of Q and P (2 bf16, 3 fp16). RW: query
// rows of a softmax warpgroup. NWG: warpgroups, each with its own rows.
template <int D_, int NT_, int RW_, int NWG_>
struct Cfg {
  static constexpr int D = D_, NT = NT_, RW = RW_, NWG = NWG_;
  static constexpr int kRows = RW * NWG;
  static constexpr int kThreads = NWG * 128 + 128;
  static constexpr int kMmaWarp = NWG * 4, kLoadWarp = NWG * 4 + 1, kQWarp = NWG * 4 + 2;
  // Who prepares an item's rows and Q: two helper warps, an item ahead of the
  // others; with several warpgroups each its own rows at the item's start,
  // where two warps took 12000 clocks for 64 rows.
  static constexpr bool kHelperQ = NWG == 1;
  static constexpr int kQParts = kHelperQ ? 2 : NWG * 4;  // warps that do
  static constexpr int kN = (NT * RW + 15) / 16 * 16;  // columns of the products
  static constexpr int kStep = NWG == 1 ? RW : 8;     // rows read from TMEM at a time
  // What an item costs a block beside its tiles, in tiles: its rows, its first
  // maximum, its result. Without it the blocks with most items were the last
  // by far (37000 clocks with one item, 61000 with four, the same tiles).
  static constexpr int kItemCost = NWG == 1 ? 2 : 4;
  static_assert(kItemCost <= kMostItemCost, "the host's bound of a share");
  // P of all warpgroups side by side: bytes of a key's row, in atoms of up to
  // 128 (three terms of 64 rows take one and a half).
  static constexpr int kPCols = NWG * kN;
  static constexpr int kPitch = kPCols <= 32 ? 32 : kPCols <= 64 ? 64 : 128;
  static constexpr int kPAtoms = (kPCols + kPitch - 1) / kPitch;
  static constexpr int kSlotBytes = kTileKeys * D;     // a K or a V tile
  static constexpr int kQBytes = kN * D;               // per warpgroup
  static constexpr int kPBytes = kTileKeys * kPitch * kPAtoms;
  static constexpr uint32_t kTmemUsed = 2u * kN * NWG;
  static constexpr uint32_t kTmemCols =
      kTmemUsed <= 32    ? 32
      : kTmemUsed <= 64  ? 64
      : kTmemUsed <= 128 ? 128
      : kTmemUsed <= 256 ? 256
                         : 512;
  static constexpr int kCtas = resident(D, RW, NWG);
  // 227 KB a block, 228 KB an SM of which each block takes 1 KB and its
  // static variables; 1 KB to align.
  static constexpr int kStatic = 2736 + 80 * kRows + 16 * NWG;
  static constexpr int kBudget = (kCtas == 1 ? 227 : (228 - kCtas) / kCtas) * 1024 - kStatic - 1024;
  // P in two buffers where four tiles of the ring still fit beside them: the
  // next one is then written while the product of this one runs.
  static constexpr int slots_with(int bufs) {
    const int n = (kBudget - NWG * 2 * kQBytes - bufs * kPBytes) / kSlotBytes;
    return n < 12 ? n : 12;
  }
  static constexpr int kPBufs = slots_with(2) >= 4 ? 2 : 1;
  static constexpr int kSlots = slots_with(kPBufs);
  static constexpr int kSmem = kSlots * kSlotBytes + NWG * 2 * kQBytes + kPBufs * kPBytes + 1024;
  // Registers: what the launch bounds give a thread, moved from the helpers
  // (loads, products, Q) to the softmax warpgroups.
  static constexpr int kRegsLaunch = 65536 / (kCtas * kThreads) / 8 * 8;
  static constexpr int kRegsHelp = NWG == 1 && kCtas == 2 ? 80 : 64;
  static constexpr int kRegsSoft = ((NWG + 1) * kRegsLaunch - kRegsHelp) / NWG / 8 * 8;
  static_assert(NWG * kRegsSoft + kRegsHelp <= (NWG + 1) * kRegsLaunch && kRegsSoft <= 255,
                "setmaxnreg must not ask for more than the block was launched with");
  static_assert(kTmemUsed <= 512 && kTmemCols * kCtas <= 512, "TMEM of the resident blocks");
  static_assert(kSlots >= 4, "a K and a V tile in use and two on their way");
  static_assert(RW == 8 || RW == 16, "rows of a warpgroup");
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
  int key0;          // first key of these items, the first of a page
  int prefix_len;    // keys of the prefix's items
  int shared_pages;  // table columns that every sequence has in row 0
  int row_tiles;     // tiles of query rows per (sequence, K/V head)
  int box;           // keys of a TMA box: min(page_size, 128)
  Divisor by_page, by_group, by_seq_rows, by_row_tiles;  // (by_seq_rows: group * seqlen_q)
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
// bytes under the 32 B, 64 B or 128 B swizzle.
template <int kPitch>
__device__ __forceinline__ uint32_t swz(int row, int col) {
  const int chunk = col >> 4;
  const int x = kPitch == 128 ? (row & 7) : kPitch == 64 ? ((row >> 1) & 3) : ((row >> 2) & 1);
  return (uint32_t)(row * kPitch + ((chunk ^ x) << 4) + (col & 15));
}

// Are all codes of row `row` of a tile of D bytes a row zero? (A swizzle moves
// pieces of 16 bytes within their row; the rows of a warp start at different ones.)
template <int D>
__device__ __forceinline__ bool zero_row(const uint8_t* tile, int row) {
  uint32_t any = 0;
#pragma unroll 1
  for (int c = 0; c < D / 16; ++c) {
    const int piece = (c + row * D / 128) % (D / 16);
    const uint4 x = *reinterpret_cast<const uint4*>(tile + row * D + piece * 16);
    any |= x.x | x.y | x.z | x.w;
  }
  return (any & 0x7f7f7f7fu) == 0;
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

// l = 2^k * x with 1 <= x < 2 for normal l; a NaN is its own x.
__device__ __forceinline__ int log2_below(float l) { return (__float_as_int(l) >> 23 & 255) - 127; }
__device__ __forceinline__ float over_log2(float l, int k) {
  return l != l ? l : __int_as_float(__float_as_int(l) - k * (1 << 23));
}
// ln(2^m l), l > 0 (or NaN): its exponent is added to m first, so that a maximum
// that is far from the largest score costs no digits.
__device__ __forceinline__ float ln_of(float m, float l) {
  const int k = log2_below(l);
  return ((m + (float)k) + log2f(over_log2(l, k))) * 0.6931471805599453f;
}

__device__ __forceinline__ float sum_of(const float4& v) { return (v.x + v.y) + (v.z + v.w); }

// P^T as operand B: rows (keys) of kPitch bytes; columns beyond them are in the
// next atom, a whole tile further on.
template <int kPitch>
__device__ __forceinline__ uint64_t desc_p(uint32_t addr) {
  uint64_t d = ptx::smem_desc_mnmajor(addr, kPitch);
  if (kPitch == 32) d = (d & ~(7ull << 61)) | (6ull << 61);  // SWIZZLE_32B
  return (d & ~(0x3FFFull << 16)) | ((uint64_t)(kTileKeys * kPitch >> 4) << 16);
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
#pragma unroll 1
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
// For what is in flight when a block ends: bounded too, but not by the caller,
// whose limit may be shorter than a copy takes.
__device__ __forceinline__ void wait_quietly(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!ptx::mbar_try_wait(bar, parity) && clock64() - t0 < kTimeout) {
  }
}

// The same for a copy that another role waits for and reports as well: until the
// block gives up.
__device__ __forceinline__ bool wait_along(uint64_t* bar, uint32_t parity, const volatile int* abort) {
  const long long t0 = clock64();
  while (!ptx::mbar_try_wait(bar, parity))
    if (*abort || clock64() - t0 > kTimeout) return false;
  return true;
}

// ----------------------------------------------------------------------- work
__device__ __forceinline__ int seq_len(const Args& a, int b) {
  if (a.prefix_mode) return a.prefix_len;
  const int len = __ldg(a.c.seqlens + b);
  return len < 0 || len > a.c.max_len ? -1 : len;
}
__device__ __forceinline__ int tiles_of(const Args& a, int len) {
  return len > a.key0 ? (len - a.key0 + kTileKeys - 1) / kTileKeys : 0;
}

// A run of key tiles t0..t1-1 of one item (sequence b, K/V head, row tile).
struct Seg {
  int b, hk, rt, t0, t1, nt, len;
  int end;  // number of the item's last unit among all
};

// Walks a block's share; every role of the block walks the same. Work is
// numbered in units: an item has `cost` for itself and then one per tile.
struct Walk {
  int b, hk, rt, off, nt, len;  // off: units of the item that lie behind
  int unit, left;
  __device__ __forceinline__ void enter(const Args& a) {
    len = seq_len(a, b);
    nt = tiles_of(a, len);
  }
  __device__ __forceinline__ bool next(const Args& a, int cost, Seg& s) {
    while (left > 0) {
      while (nt == 0) {
        ++b;
        enter(a);
      }
      s.b = b;
      s.hk = hk;
      s.rt = rt;
      s.nt = nt;
      s.len = len;
      s.end = unit - off + cost + nt - 1;
      s.t0 = max(0, off - cost);
      const int take = min(cost + nt - off, left);
      off += take;
      unit += take;
      left -= take;
      s.t1 = max(0, off - cost);
      if (off == cost + nt) {
        off = 0;
        if (++rt == a.row_tiles) {
          rt = 0;
          if (++hk == a.c.heads_kv) {
            hk = 0;
            ++b;
            if (left > 0) enter(a);
          }
        }
      }
      if (s.t1 > s.t0) return true;
    }
    return false;
  }
};

// Shares of `total` units over `n` blocks: the first total % n have one more.
struct Shares {
  int size, more;
  __device__ __forceinline__ Shares(int total, int n) : size(total / n), more(total - size * n) {}
  __device__ __forceinline__ int begin(int c) const { return c * size + min(c, more); }
  __device__ __forceinline__ int block_of(int unit) const {
    const int wide = more * (size + 1);
    return unit < wide ? unit / (size + 1) : more + (unit - wide) / size;
  }
};

__device__ __forceinline__ int page_of(const Args& a, int key) {
  return a.by_page.div(key);
}

constexpr int kExpTiles = 8;  // ring of exponent bytes: tiles in flight and two more

template <class C>
struct __align__(16) Shared {
  uint8_t exps[kExpTiles][2][kTileKeys];  // of K and V
  uint64_t kv_full[C::kSlots];
  uint64_t kv_empty[C::kSlots];
  uint64_t e_full[kExpTiles];
  uint64_t q_full[2];        // Q and row data of an item, two items in turn
  uint64_t q_free[2];
  uint64_t s_full;           // S^T of all warpgroups in TMEM
  uint64_t s_free;           // read by their warps, and the tile's exponents
  // P^T in shared memory (and O^T rescaled), tiles in turn: the softmax may be
  // done with tile n + 1 before the products have looked for tile n, but not
  // with tile n + 2, whose scores are issued behind the values of tile n.
  uint64_t p_full[2];
  uint64_t o_done[2];        // O^T += V^T P^T complete, tiles in turn
  uint64_t drain;
  uint32_t tmem;
  int abort;
  int again;                 // kRef does not serve an exponent of V
  Walk start;                // where the block's share begins
  struct __align__(16) Rows {  // of an item; read four at a time
    float mul[C::kRows];     // scale * log2(e) * the power of two of the row of Q
    int row_id[C::kRows];    // (b * heads + h) * seqlen_q + i; -1: no such row
    int lim[C::kRows];       // keys that the row sees
    long long off[C::kRows]; // where a whole row's result goes, in elements
    int all_see[kMostWarps]; // keys that all rows of a warp see
    Seg seg;                 // the item, and whether it is the block's last
    int last;                // (written and read where helpers prepare it)
  } rows[2];
  struct Group {
    float neg_m[C::RW];      // minus the running maxima
    float step[C::RW];       // and what the last rise added to that
    float4 sum[C::RW];       // the four warps' sums of a row
    float4 top[C::RW];       // and maxima of a tile
    uint32_t solid;          // a byte of each warp: has its part of the tile rows that are not zeros?
    uint32_t pad[3];
  } g[C::NWG];
  static_assert(sizeof(Rows) % 16 == 0 && sizeof(Group) % 16 == 0, "read four at a time");
  static_assert(C::kSlots / 2 + 2 <= kExpTiles,
                "a tile's exponents are read before their place is used again");
};

// Row j of item rows (K/V head hk; sequence b unless the items are the
// prefix's): its sequence, head and query.
struct Row {
  int b, h, i;
  __device__ __forceinline__ Row(const Args& a, int seq, int hk, int j) {
    b = seq;
    if (a.prefix_mode) {
      b = a.by_seq_rows.div(j);
      j -= b * a.by_seq_rows.d;
    }
    i = a.by_group.div(j);
    h = hk * a.group + j - i * a.group;
  }
};

// Sums over the warp of N values per lane: lane l has that of value
// l / (32 / N). Every step halves the values a lane keeps.
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N]) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int half = N / 2, o = 16; half; half >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float give = up ? v[i] : v[i + half], keep = up ? v[i + half] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
#pragma unroll
  for (int o = 16 / N; o; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}

// Row data of an item and its Q as terms, K-major: rows first..first+ROWS-1 of
// its tile by WARPS warps, of which this one is number `me`. Rows beyond the
// last, up to a whole step, are made zero: they are computed with.
template <class C, bool kBf16, int ROWS, int WARPS, class Rows>
__device__ __forceinline__ void prepare_rows(const Args& a, const Seg& s, Rows& rw, uint8_t* q_item,
                                             int first, int me) {
  constexpr int D = C::D, NT = C::NT, RW = C::RW;
  constexpr int kLanes = D / 8, kPer = 32 / kLanes;  // lanes of a row; rows of a warp at a time
  constexpr int kShare = ROWS / WARPS / kPer;
  constexpr int kMost = C::kHelperQ && C::kRegsHelp < 80 ? 2 : 4;  // loads in flight
  constexpr int kBatch = kShare < kMost ? kShare : kMost;
  static_assert(ROWS % (kPer * kBatch * WARPS) == 0, "whole batches");
  const int lane = threadIdx.x % 32, cl = lane % kLanes;
  const int rows = a.seqlen_q * a.group * (a.prefix_mode ? a.c.batch : 1);
  const int row0 = s.rt * C::kRows + first, used = min(ROWS, rows - row0);
  const int filled = (used + C::kStep - 1) / C::kStep * C::kStep;
  uint4 xs[kBatch];
  auto ask = [&](int r0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int r = r0 + u * kPer + lane / kLanes;
      xs[u] = make_uint4(0, 0, 0, 0);
      if (r < used) {
        const Row row(a, s.b, s.hk, row0 + r);
        xs[u] = __ldg(reinterpret_cast<const uint4*>(
                          a.q + 2 * (row.b * a.q_sb + row.h * a.q_sh + row.i * a.q_ss)) + cl);
      }
    }
  };
  ask(me * kPer * kBatch);  // on their way while the row data is made
  int see = s.len;
#pragma unroll 1
  for (int r = me * 32 + lane; r < ROWS; r += 32 * WARPS) {
    int lim = s.len, id = -1;
    long long off = 0;
    if (r < used) {
      const Row row(a, s.b, s.hk, row0 + r);
      int len = s.len;
      if (a.prefix_mode) {
        len = __ldg(a.c.seqlens + row.b);
        if (len < 0 || len > a.c.max_len) len = 0;  // refused: its rows are not joined
      }
      lim = max(0, min(s.len, len - a.seqlen_q + row.i + 1));
      id = (row.b * a.heads + row.h) * a.seqlen_q + row.i;
      off = a.own_rows ? row.b * a.o_sb + row.h * a.o_sh + row.i * a.o_ss : (long long)id * D;
    }
    rw.lim[first + r] = lim;
    rw.row_id[first + r] = id;
    rw.off[first + r] = off;
    see = min(see, lim);
  }
  see = __reduce_min_sync(0xffffffffu, see);
  if (lane == 0) rw.all_see[first / ROWS * WARPS + me] = see;
#pragma unroll 1
  for (int r0 = me * kPer * kBatch; r0 < filled; r0 += WARPS * kPer * kBatch) {
    // Stage by stage over the batch: a warp by itself is as fast as its
    // chains are side by side.
    uint32_t top[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const uint32_t m = __vmaxu2(__vmaxu2(xs[u].x & 0x7fff7fffu, xs[u].y & 0x7fff7fffu),
                                  __vmaxu2(xs[u].z & 0x7fff7fffu, xs[u].w & 0x7fff7fffu));
      top[u] = max(m & 0xffffu, m >> 16);
    }
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        top[u] = max(top[u], __shfl_xor_sync(0xffffffffu, top[u], o));
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int r = r0 + u * kPer + lane / kLanes;
      const uint32_t m = top[u];
      const bool fine = m < (kBf16 ? 0x7f80u : 0x7c00u);
      const uint32_t bits =
          kBf16 ? m << 16
                : __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
      // 2^(7 - e) with 2^e <= max < 2^(e + 1); rows below 2^-100 (bf16) are held to
      // 2^-121, as rows of 2^-100 are.
      const int e = m == 0 ? 7 : max((int)(bits >> 23) - 127, -100);
      if (cl == 0)
        rw.mul[first + r] = fine ? a.scale_log2 * __uint_as_float((uint32_t)(127 - 7 + e) << 23)
                         : __int_as_float(0x7fc00000);
      const float f = fine ? __uint_as_float((uint32_t)(127 + 7 - e) << 23) : 0.f;
      auto scale2 = [&](uint32_t word) -> uint32_t {
        float2 v;
        if (kBf16)
          v = make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
        else
          v = __half22float2(*reinterpret_cast<const __half2*>(&word));
        return fine ? h2(v.x * f, v.y * f) : 0u;
      };
      xs[u] = make_uint4(scale2(xs[u].x), scale2(xs[u].y), scale2(xs[u].z), scale2(xs[u].w));
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int r = r0 + u * kPer + lane / kLanes;
        const uint16_t e0 = e4m3x2_of_h2(xs[u].x), e1 = e4m3x2_of_h2(xs[u].y),
                       e2 = e4m3x2_of_h2(xs[u].z), e3 = e4m3x2_of_h2(xs[u].w);
        *reinterpret_cast<uint2*>(q_item + (first + r) / RW * C::kQBytes +
                                  swz<D>(t * RW + r % RW, cl * 8)) =
            make_uint2((uint32_t)e0 | ((uint32_t)e1 << 16), (uint32_t)e2 | ((uint32_t)e3 << 16));
        if (t + 1 < NT)
          xs[u] = make_uint4(rest(xs[u].x, e0), rest(xs[u].y, e1), rest(xs[u].z, e2),
                             rest(xs[u].w, e3));
      }
    }
    ask(r0 + WARPS * kPer * kBatch);
  }
}

// The values of four codes.
__device__ __forceinline__ void floats_of(uint32_t w, float (&x)[4]) {
  const uint32_t h0 = ptx::cvt_e4m3x2_to_f16x2((uint16_t)w),
                 h1 = ptx::cvt_e4m3x2_to_f16x2((uint16_t)(w >> 16));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0)),
               b = __half22float2(*reinterpret_cast<const __half2*>(&h1));
  x[0] = a.x;
  x[1] = a.y;
  x[2] = b.x;
  x[3] = b.y;
}

// A block's share once more, by its softmax warps, in fp32 and straight from the
// cache: for values so large or small that kRef does not serve them, or so far
// apart. R rows at a time; a warp takes every W-th run of 32
// keys, a lane a key for the scores and D / 32 columns for the values. The
// maximum of s is the weights' reference, that of s + e the sum of values', so
// neither leaves the range of fp32. A call whose every share is computed again
// takes six to eight times as long (64 sequences of up to 16384 keys 1170 us), 15
// times behind a shared prefix. Kept apart from the loop over tiles: as a branch
// of it, with a second exponential for P, it cost every call 10 to 17 %.
template <class C, bool kBf16>
__device__ __forceinline__ void share_again(const Args& a, Walk walk, float* scratch) {
  // (Two rows in the blocks of which three share an SM: four spilled there, which
  // the loop over tiles paid for as well.)
  constexpr int D = C::D, W = C::NWG * 4, R = C::kCtas == 3 ? 2 : 4, V = D / 32;
  static_assert((R * D + 3 * W * R + W * R * D) * 4 <= C::kSlots * C::kSlotBytes, "scratch in the ring");
  float* const q_s = scratch;           // [R][D]
  float* const ms_s = q_s + R * D;      // [W][R] of each warp: maximum of s,
  float* const me_s = ms_s + W * R;     // of s + e,
  float* const l_s = me_s + W * R;      // sum,
  float* const o_s = l_s + W * R;       // [W][R][D] and sums of values
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const kv::CacheView& c = a.c;
  const int rows = a.seqlen_q * a.group * (a.prefix_mode ? c.batch : 1);
  Seg s;
  for (int k = 0; walk.next(a, C::kItemCost, s); ++k) {
    const int used = min(C::kRows, rows - s.rt * C::kRows);
    const bool whole = s.t0 == 0 && s.t1 == s.nt;
    const int part = 2 * blockIdx.x + (k > 0 ? 1 : 0);
    const int first = a.key0 + s.t0 * kTileKeys, last = min(s.len, a.key0 + s.t1 * kTileKeys);
    const int* const table = c.table + (a.prefix_mode ? 0 : s.b) * c.table_stride;
#pragma unroll 1
    for (int r0 = 0; r0 < used; r0 += R) {
      ptx::named_barrier_sync(kAgainBar, W * 32);  // the scratch is free
#pragma unroll 1
      for (int i = threadIdx.x; i < R * D; i += W * 32) {
        const int r = r0 + i / D;
        float x = 0.f;
        if (r < used) {
          const Row row(a, s.b, s.hk, s.rt * C::kRows + r);
          const unsigned short w = __ldg(reinterpret_cast<const unsigned short*>(a.q) +
                                         row.b * a.q_sb + row.h * a.q_sh + row.i * a.q_ss + i % D);
          x = kBf16 ? __uint_as_float((uint32_t)w << 16) : __half2float(__ushort_as_half(w));
          // 2^20 less: D products of the largest bf16 with codes stay in fp32. A row
          // with an infinity is NaN, as it is on the tensor cores.
          x = fabsf(x) < INFINITY ? x * 0x1p-20f : __int_as_float(0x7fc00000);
        }
        q_s[i] = x;
      }
      int lim[R];
      float ms[R], me[R], l[R], o[R][V];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        lim[r] = 0;
        if (r0 + r < used) {
          const Row row(a, s.b, s.hk, s.rt * C::kRows + r0 + r);
          const int len = a.prefix_mode ? __ldg(c.seqlens + row.b) : s.len;
          if (len >= 0 && len <= c.max_len) lim[r] = min(last, len - a.seqlen_q + row.i + 1);
        }
        ms[r] = me[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) o[r][v] = 0.f;
      }
      ptx::named_barrier_sync(kAgainBar, W * 32);
#pragma unroll 1
      for (int key0 = first + warp * 32; key0 < last; key0 += W * 32) {
        const int key = key0 + lane;
        const uint8_t *kr = nullptr, *vr = nullptr;
        int kb = kv::kExpNan, vb = kv::kExpNan;
        if (key < last) {
          const int col = page_of(a, key), slot = key - col * c.page_size;
          const long long page = __ldg((col < a.shared_pages ? c.table : table) + col);
          if (page >= 0 && page < c.num_pages) {
            kr = c.k + page * c.k_sp + s.hk * c.k_sh + slot * c.k_ss;
            vr = c.v + page * c.v_sp + s.hk * c.v_sh + slot * c.v_ss;
            kb = c.k_exp[page * c.ke_sp + s.hk * c.ke_sh + slot];
            vb = c.v_exp[page * c.ve_sp + s.hk * c.ve_sh + slot];
          }
        }
        float y[R];
#pragma unroll
        for (int r = 0; r < R; ++r) y[r] = 0.f;
        if (kr) {
#pragma unroll 1
          for (int d = 0; d < D; d += 16) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(kr + d));
            const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float f[4];
              floats_of(words[i], f);
#pragma unroll
              for (int r = 0; r < R; ++r) {
                const float4 q4 = *reinterpret_cast<const float4*>(q_s + r * D + d + 4 * i);
                y[r] = fmaf(q4.x, f[0], fmaf(q4.y, f[1], fmaf(q4.z, f[2], fmaf(q4.w, f[3], y[r]))));
              }
            }
          }
        }
        const float kf = kv::exp_factor(kb), e = (float)(vb - kv::kExpBias);
        uint32_t any = 1;
        if (vr && vb == kv::kExpBias) {
          any = 0;
#pragma unroll 1
          for (int d = 0; d < D; d += 4)
            any |= __ldg(reinterpret_cast<const uint32_t*>(vr + d)) & 0x7f7f7f7fu;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float sc = key < lim[r] ? y[r] * kf * (a.scale_log2 * 0x1p20f) : -INFINITY;
          const float t = any && vb != kv::kExpNan ? sc + e : -INFINITY;
          const float m_new = fmaxf(ms[r], warp_max(sc)), e_new = fmaxf(me[r], warp_max(t));
          const float m_use = m_new == -INFINITY ? 0.f : m_new, e_use = e_new == -INFINITY ? 0.f : e_new;
          l[r] = l[r] * ptx::ex2(ms[r] - m_use) + ptx::ex2(sc - m_use);
          const float f = ptx::ex2(me[r] - e_use);
#pragma unroll
          for (int v = 0; v < V; ++v) o[r][v] *= f;
          y[r] = sc == -INFINITY         ? 0.f
                 : vb == kv::kExpNan ? __int_as_float(0x7fc00000)
                                     : ptx::ex2(t - e_use);
          ms[r] = m_new;
          me[r] = e_new;
        }
#pragma unroll 4
        for (int kk = 0; kk < 32; ++kk) {
          const uint8_t* const row =
              reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, (unsigned long long)vr, kk));
          uint32_t w = 0;
          if (row)
            w = V == 4 ? __ldg(reinterpret_cast<const uint32_t*>(row) + lane)
                       : __ldg(reinterpret_cast<const unsigned short*>(row) + lane);
          float x[4];
          floats_of(w, x);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float yr = __shfl_sync(0xffffffffu, y[r], kk);
#pragma unroll
            for (int v = 0; v < V; ++v) o[r][v] = fmaf(yr, x[v], o[r][v]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 16; i; i >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], i);
        const int at = warp * R + r;
        if (lane == 0) {
          ms_s[at] = ms[r];
          me_s[at] = me[r];
          l_s[at] = l[r];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) o_s[at * D + lane * V + v] = o[r][v];
      }
      ptx::named_barrier_sync(kAgainBar, W * 32);
      const int r = r0 + warp;
      if (warp < R && r < used) {  // a warp joins a row
        float m = -INFINITY, e = -INFINITY, sum = 0.f, x[V];
        for (int w = 0; w < W; ++w) {
          m = fmaxf(m, ms_s[w * R + warp]);
          e = fmaxf(e, me_s[w * R + warp]);
        }
        const float m_use = m == -INFINITY ? 0.f : m, e_use = e == -INFINITY ? 0.f : e;
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = 0.f;
        for (int w = 0; w < W; ++w) {
          const int at = w * R + warp;
          sum = fmaf(ptx::ex2(ms_s[at] - m_use), l_s[at], sum);
          const float f = ptx::ex2(me_s[at] - e_use);
#pragma unroll
          for (int v = 0; v < V; ++v) x[v] = fmaf(f, o_s[at * D + lane * V + v], x[v]);
        }
        // times 2^(e - m), in two steps for the range of fp32
        const float by = e == -INFINITY ? 0.f : e - m_use, here = fminf(fmaxf(by, -100.f), 100.f);
        const float f0 = sum == 0.f ? 0.f : ptx::ex2(here) / sum, f1 = ptx::ex2(by - here);
        const float top = sum == 0.f ? -INFINITY : m;
        const Row row(a, s.b, s.hk, s.rt * C::kRows + r);
        const long long id = (row.b * a.heads + row.h) * a.seqlen_q + row.i;
        const long long at = (long long)part * C::kRows + r;
        if (lane == 0) {
          if (!whole)
            a.part_ml[at] = make_float2(top, sum);
          else if (!a.own_rows)
            a.full_ml[id] = make_float2(top, sum);
          else if (a.lse)
            a.lse[id] = sum == 0.f ? -INFINITY : ln_of(top, sum);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float out = x[v] * f0 * f1;
          // A part that is to be weighted stays finite: bf16's largest is 2^128 as a
          // code and a power of two, just above fp32's.
          if (!(whole && a.own_rows) && fabsf(out) == INFINITY) out = copysignf(FLT_MAX, out);
          const int d = lane * V + v;
          if (!whole)
            a.part_o[at * D + d] = out;
          else if (!a.own_rows)
            a.full_o[id * D + d] = out;
          else if (kBf16)
            reinterpret_cast<__nv_bfloat16*>(a.o)[row.b * a.o_sb + row.h * a.o_sh + row.i * a.o_ss + d] =
                __float2bfloat16(out);
          else
            reinterpret_cast<__half*>(a.o)[row.b * a.o_sb + row.h * a.o_sh + row.i * a.o_ss + d] =
                __float2half(out);
        }
      }
    }
  }
}

template <class C, bool kBf16>
__global__ void __launch_bounds__(C::kThreads, C::kCtas)
    decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const Args a) {
  constexpr int D = C::D, NT = C::NT, RW = C::RW, NS = C::kSlots;
  static_assert(sizeof(Shared<C>) <= C::kStatic, "shared memory budget");
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared<C> sh;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int G = gridDim.x, cta = blockIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == C::kLoadWarp && lane == 0) {
    ptx::tma_prefetch_desc(&tm_k);
    ptx::tma_prefetch_desc(&tm_v);
  }
  if (warp == 0) {
    for (int i = lane; i < NS; i += 32) {
      ptx::mbar_init(&sh.kv_full[i], 1);
      ptx::mbar_init(&sh.kv_empty[i], 1);
    }
    if (lane < kExpTiles) ptx::mbar_init(&sh.e_full[lane], 32);
    if (lane < 2) {
      ptx::mbar_init(&sh.q_full[lane], C::kQParts);
      ptx::mbar_init(&sh.q_free[lane], C::NWG * 4);
      ptx::mbar_init(&sh.p_full[lane], C::NWG * 4);
      ptx::mbar_init(&sh.o_done[lane], 1);
    }
    if (lane == 0) {
      ptx::mbar_init(&sh.s_full, 1);
      ptx::mbar_init(&sh.s_free, C::NWG * 4);
      ptx::mbar_init(&sh.drain, 1);
      sh.abort = sh.again = 0;
    }
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }

  // ------------------------------------------------- this block's share
  // Every warp finds it for itself: lane i counts the units of a run of
  // sequences, a scan says how many come before. (The host has checked that
  // they number less than 2^31.)
  const int nseq = a.prefix_mode ? 1 : a.c.batch;
  const int chunk = (nseq + 31) / 32;
  const int s0 = min(nseq, lane * chunk), s1 = min(nseq, s0 + chunk);
  const int per = a.c.heads_kv * a.row_tiles;
  int mine = 0;
#pragma unroll 4
  for (int b = s0; b < s1; ++b) {
    const int len = seq_len(a, b);
    if (len < 0 && cta == 0 && warp == 0 && a.c.status)
      atomicOr(a.c.status, FA8_DEVERR_VARLEN_RANGE);
    const int nt = tiles_of(a, len);
    mine += nt > 0 ? per * (C::kItemCost + nt) : 0;
  }
  if (warp == C::kMmaWarp) {
    ptx::tmem_alloc(&sh.tmem, C::kTmemCols);
    ptx::tmem_relinquish();
  }
  int upto = mine;  // inclusive scan
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  const int total = __shfl_sync(0xffffffffu, upto, 31);
  const int active = min(G, total);  // blocks with a share
  const Shares shares(total, max(active, 1));
  const int u0 = cta < active ? shares.begin(cta) : 0;
  const int u1 = cta < active ? shares.begin(cta + 1) : 0;
  Walk walk;
  walk.left = u1 - u0;
  walk.unit = u0;
  {
    const uint32_t here = __ballot_sync(0xffffffffu, u0 >= upto - mine && u0 < upto);
    const int src = __ffs(here) - 1;  // the lane in whose sequences unit u0 is
    if (u0 < u1) {
      int at = __shfl_sync(0xffffffffu, upto - mine, src);
      for (walk.b = __shfl_sync(0xffffffffu, s0, src);; ++walk.b) {
        walk.enter(a);
        if (walk.nt == 0) continue;
        const int n = per * (C::kItemCost + walk.nt);
        if (u0 < at + n) break;
        at += n;
      }
      const int each = C::kItemCost + walk.nt, item = (u0 - at) / each;
      walk.off = u0 - at - item * each;
      walk.hk = a.by_row_tiles.div(item);
      walk.rt = item - walk.hk * a.row_tiles;
    }
  }

  if (threadIdx.x == 0) sh.start = walk;

  // Sequences without a key among these items have no tile and no block of
  // their own: their rows (items) are filled in by block b mod G.
  auto fill_empty = [&](int first, int step) {
    if (a.prefix_mode) return;
    for (int b = cta; b < a.c.batch; b += G) {
      const int len = seq_len(a, b);
      if (len < 0 || tiles_of(a, len) > 0) continue;
      if (a.own_rows) {
        const int n = a.heads * a.seqlen_q;
        const int piece = first % (D / 8);
        for (int row = first / (D / 8); row < n; row += step / (D / 8)) {
          const int h = row / a.seqlen_q, i = row - h * a.seqlen_q;
          reinterpret_cast<uint4*>(a.o + 2 * (b * a.o_sb + h * a.o_sh + i * a.o_ss))[piece] =
              make_uint4(0, 0, 0, 0);
          if (a.lse && piece == 0) a.lse[(long long)b * n + row] = -INFINITY;
        }
      } else {
        for (int j = first; j < per; j += step)
          a.item[(long long)b * per + j] = make_int4(0, 0, 0, kItemEmpty);
      }
    }
  };
  // Says where the parts of the block's item k are, if it begins here: from
  // this block to that of its last tile. One thread does, from the start on.
  auto no_parts = [&]() {
    if (a.own_rows) a.seg[cta] = make_int4(-1, 0, 0, 0);
  };
  auto say_parts = [&](const Seg& s, int k) {
    const bool whole = s.t1 == s.nt;
    if (s.t0 > 0 || (a.own_rows && whole)) return;
    const int part = 2 * cta + (k > 0 ? 1 : 0), row = s.hk * a.row_tiles + s.rt;
    const int last = whole ? cta : shares.block_of(s.end);
    if (a.own_rows)
      a.seg[cta] = make_int4(last, s.b, row, part);
    else
      a.item[(long long)s.b * per + row] =
          make_int4(cta, last, part, whole ? kItemFull : kItemParts);
  };
  // Barriers and TMEM are there for all. Every role comes here when it has
  // asked for its first data.
  auto block_sync = [&]() {
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
  };
  auto end_sync = [&]() {
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
  };
  Seg s;
  bool more = walk.next(a, C::kItemCost, s);
  if (!more) {  // no share, or one that ends before its item's first tile
    block_sync();
    if (warp == C::kMmaWarp) ptx::tmem_dealloc(sh.tmem, C::kTmemCols);
    fill_empty(threadIdx.x, C::kThreads);
    if (threadIdx.x == 0) no_parts();
    if (a.early) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  // Ring of K and V tiles | P | Q of two items.
  uint8_t* const p_tiles = smem + NS * C::kSlotBytes;
  uint8_t* const q_tiles = p_tiles + C::kPBufs * C::kPBytes;
  const Waiter wait{&sh.abort, a.c.status, a.timeout};
  if (warp >= C::kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsHelp));
    if (warp == C::kLoadWarp) {
      // ------------------------------------------------------------ TMA producer
      // Lane l brings piece l (box keys of one page) of a K and of a V tile.
      // Ring item 2n is K of the block's tile n, 2n + 1 its V. Lanes 0-15 bring
      // the tile's exponent bytes, 16 keys of K or V each.
      const int pieces = kTileKeys / a.box;
      const uint64_t policy = a.row_tiles > 1 ? ptx::policy_evict_last() : ptx::policy_evict_first();
      const bool is_v = lane >= 8;
      const int e_key = (lane & 7) * 16, e_piece = e_key / a.box;
      const uint8_t* const exps = is_v ? a.c.v_exp : a.c.k_exp;
      const long long e_sp = is_v ? a.c.ve_sp : a.c.ke_sp, e_sh = is_v ? a.c.ve_sh : a.c.ke_sh;
      int n = 0, issued = 0;
      bool ok = true;
      for (bool first = true; ok && more; more = walk.next(a, C::kItemCost, s), first = false) {
        const int* table = a.c.table + (a.prefix_mode ? 0 : s.b) * a.c.table_stride;
        // Table entries of the item's next 32 pieces, one a lane: one load for 4
        // to 32 tiles, asked for a batch ahead.
        auto entries = [&](int piece) {
          const int key = a.key0 + s.t0 * kTileKeys + (piece + lane) * a.box;
          if (key >= min(s.len, a.key0 + s.t1 * kTileKeys)) return 0;
          const int col = page_of(a, key);
          return __ldg((col < a.shared_pages ? a.c.table : table) + col);
        };
        int cur = entries(0), next = entries(32), piece = 0;
        if (first) block_sync();
        for (int t = s.t0; t < s.t1; ++t, ++n, piece += pieces) {
          if (piece == 32) {
            piece = 0;
            cur = next;
            next = entries((t - s.t0) * pieces + 32);
          }
          const int page = __shfl_sync(0xffffffffu, cur, (piece + lane) & 31);
          const int key0 = a.key0 + t * kTileKeys, key = key0 + lane * a.box;
          const bool have = lane < pieces && key < s.len;
          // A page outside the cache: coordinates that read as zeros, exponents
          // that say NaN.
          const bool outside = page < 0 || page >= a.c.num_pages;
          if (have && outside && a.c.status) atomicOr(a.c.status, FA8_DEVERR_PAGE_RANGE);
          const int coord = outside ? 0x7fffffff : page;
          const int slot = key - page_of(a, key) * a.c.page_size;
          const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, have)) * a.box * D;
          const int e_coord = __shfl_sync(0xffffffffu, coord, e_piece);
          const int e_slot = __shfl_sync(0xffffffffu, slot, e_piece) + e_key - e_piece * a.box;
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
            if (v == 0) {
              // K's place is free: the scores of kSlots / 2 tiles ago are done,
              // so the tile before that has been read, exponents included.
              uint8_t* const dst = &sh.exps[n % kExpTiles][is_v][e_key];
              uint64_t* const bar = &sh.e_full[n % kExpTiles];
              const bool mine = lane < 16 && key0 + e_key < s.len;
              if (mine && e_coord == 0x7fffffff) {
                *reinterpret_cast<uint4*>(dst) = make_uint4(~0u, ~0u, ~0u, ~0u);
                ptx::mbar_arrive(bar);
              } else {
                if (mine)
                  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(dst)),
                               "l"(exps + e_coord * e_sp + s.hk * e_sh + e_slot)
                               : "memory");
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                                 ptx::smem_u32(bar))
                             : "memory");
              }
            }
          }
          if (!ok) break;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (lane == 0) {
        // Copies in flight land before the block ends, whoever gave up waiting:
        // a share that fits the ring never makes this warp wait, so it does not
        // learn of it. When nobody did they have landed, and this is at once.
        for (int i = max(0, issued - NS); i < issued; ++i)
          wait_quietly(&sh.kv_full[i % NS], (i / NS) & 1);
      }
    } else if (warp >= C::kQWarp && !C::kHelperQ) {
      block_sync();
    } else if (warp >= C::kQWarp) {
      // ------------------------------------------------------------ rows and Q
      const int me = warp - C::kQWarp;
      block_sync();
      const bool speaks = me == 0 && lane == 0;
      if (speaks) no_parts();
      for (int k = 0; more; ++k) {
        const int buf = k & 1;
        if (k >= 2 && !wait.warp(&sh.q_free[buf], ((k >> 1) - 1) & 1)) break;
        prepare_rows<C, kBf16, C::kRows, 2>(a, s, sh.rows[buf], q_tiles + buf * C::NWG * C::kQBytes, 0,
                                            me);
        if (speaks) {
          sh.rows[buf].seg = s;
          say_parts(s, k);
        }
        more = walk.next(a, C::kItemCost, s);
        if (speaks) sh.rows[buf].last = !more;
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sh.q_full[buf]);
      }
    } else if (warp == C::kMmaWarp) {
      block_sync();
      if (lane == 0) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t tmem = sh.tmem;
        const uint32_t ring = ptx::smem_u32(smem), pb = ptx::smem_u32(p_tiles),
                       qb = ptx::smem_u32(q_tiles);
        // One product for all warpgroups: an instruction costs the issuing thread
        // some 100 clocks whatever its N (one product of values per warpgroup
        // made this thread the slowest of all: 5000 clocks a tile of 64 rows).
        constexpr uint32_t idesc_s = ptx::idesc_e4m3_f32(128, C::NWG * C::kN);
        constexpr uint32_t idesc_o = idesc_tt(128, C::NWG * C::kN);
        bool ok = true;
        auto scores = [&](int n, int k, bool first) {  // S^T of tile n, in item k
          const int i = 2 * n, st = i % NS;
          if (first) ok = wait(&sh.q_full[k & 1], (k >> 1) & 1);
          ok = ok && wait(&sh.kv_full[st], (i / NS) & 1);
          if (n > 0) ok = ok && wait(&sh.s_free, (n - 1) & 1);
          if (!ok) return;
          ptx::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 32; ++kk)
            ptx::umma_f8(tmem, ptx::smem_desc_kmajor(ring + st * C::kSlotBytes + kk * 32, D),
                         ptx::smem_desc_kmajor(qb + (k & 1) * C::NWG * C::kQBytes + kk * 32, D), idesc_s,
                         kk > 0 ? 1u : 0u);
          ptx::umma_commit(&sh.s_full);
          ptx::umma_commit(&sh.kv_empty[st]);
        };
        auto values = [&](int n, bool first) {  // O^T += V^T P^T of tile n
          const int i = 2 * n + 1, st = i % NS;
          ok = wait(&sh.kv_full[st], (i / NS) & 1);
          ok = ok && wait(&sh.p_full[n & 1], (n >> 1) & 1);
          if (!ok) return;
          ptx::tc_fence_after();
          const uint32_t p = pb + n % C::kPBufs * C::kPBytes;
#pragma unroll
          for (int kk = 0; kk < kTileKeys / 32; ++kk)
            ptx::umma_f8(tmem + C::NWG * C::kN, desc_v<D>(ring + st * C::kSlotBytes + kk * 32 * D),
                         desc_p<C::kPitch>(p + kk * 32 * C::kPitch), idesc_o,
                         first && kk == 0 ? 0u : 1u);
          ptx::umma_commit(&sh.o_done[n & 1]);
          ptx::umma_commit(&sh.kv_empty[st]);
        };
        // The scores of the next tile, be it the next item's first, are issued
        // before this tile's values: they are ready when its softmax is done.
        int n = 0;
        scores(0, 0, true);
        for (int k = 0; ok && more; ++k) {
          const Seg& now = C::kHelperQ ? sh.rows[k & 1].seg : s;
          const int count = now.t1 - now.t0;
          for (int j = 0; ok && j < count; ++j, ++n) {
            if (j + 1 < count) {
              scores(n + 1, k, false);
            } else if (C::kHelperQ) {
              more = !sh.rows[k & 1].last;
              if (more) scores(n + 1, k + 1, true);
            }
            if (ok) values(n, j == 0);
          }
          // Warpgroups that prepare their rows themselves do so when the item
          // before is done.
          if (!C::kHelperQ) {
            more = walk.next(a, C::kItemCost, s);
            if (ok && more) scores(n, k + 1, true);
          }
        }
        ptx::umma_commit(&sh.drain);
        wait_quietly(&sh.drain, 0);
      }
    }
    end_sync();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoft));
    // --------------------------------------------------------------- softmax
    block_sync();
    fill_empty(threadIdx.x, C::NWG * 128);  // (nothing to do yet)
    const uint32_t tmem = sh.tmem;
    const int w = warp / 4, wq = warp % 4, tid = threadIdx.x % 128;
    auto& g = sh.g[w];
    bool ok = true;
    // The warpgroup's barrier: does any thread say yes?
    auto any_of = [&](bool yes) -> bool {
      uint32_t any;
      asm volatile(
          "{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n"
          " barrier.cta.red.or.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
          : "=r"(any)
          : "r"(1 + w), "r"((uint32_t)yes)
          : "memory");
      return any != 0;
    };
    const uint32_t lanes = (uint32_t)(wq * 32) << 16;
    const uint32_t col_s = tmem + w * C::kN + lanes, col_o = tmem + (C::NWG + w) * C::kN + lanes;
    int n = 0, k = 0;
    // A warp whose wait gave up goes on to the next barrier, and all four
    // leave there together.
    bool left = false;
    if (!C::kHelperQ && threadIdx.x == 0) no_parts();
    for (;; ++k) {
      const auto& rw = sh.rows[k & 1];
      bool last = false;
      if constexpr (C::kHelperQ) {
        ok = ok && wait.warp(&sh.q_full[k & 1], (k >> 1) & 1);
        if (!ok) {  // the two barriers where the other warps leave
          any_of(true);
          any_of(true);
          break;
        }
        s = rw.seg;
        last = rw.last;
      } else {
        prepare_rows<C, kBf16, RW, 4>(a, s, sh.rows[k & 1],
                                      q_tiles + (k & 1) * C::NWG * C::kQBytes, w * RW, wq);
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sh.q_full[k & 1]);
        if (threadIdx.x == 0) say_parts(s, k);
        ok = ok && wait.warp(&sh.q_full[k & 1], (k >> 1) & 1);
      }
      // Keys that all this warpgroup's rows see.
      const int all_see = C::kHelperQ ? min(rw.all_see[0], rw.all_see[1]) : rw.all_see[4 * w];
      // Rows that exist: steps without any are not computed.
      const int rows = a.seqlen_q * a.group * (a.prefix_mode ? a.c.batch : 1);
      const int used = min(RW, rows - s.rt * C::kRows - w * RW);
      uint64_t l2[RW / 2];  // sums of p over this thread's keys, pairs of rows
#pragma unroll
      for (int r = 0; r < RW / 2; ++r) l2[r] = 0;
      // Running maximum of row `lane`. A row that sees any of this block's keys
      // of the item sees some of the first tile: that one sets it. As long as no
      // value row but zeros has been met (`bare`) the next tile is looked at too.
      float m_lane = 0.f;
      bool bare = true;
      if (lane < RW) g.neg_m[lane] = 0.f;  // (every warp writes the same)
      __syncwarp();
      for (int t = s.t0; t < s.t1; ++t, ++n) {
        const int first_key = a.key0 + t * kTileKeys, key = first_key + tid;
        // Every key of the tile seen by every row? This one by any?
        const bool plain = first_key + kTileKeys <= all_see, dead = key >= s.len;
        ok = ok && wait.warp(&sh.e_full[n % kExpTiles], (n / kExpTiles) & 1);
        const int kb = sh.exps[n % kExpTiles][0][tid], vb = sh.exps[n % kExpTiles][1][tid];
        const float kf = kv::exp_factor(kb);
        const bool first = t == s.t0, v_nan = !dead && vb == kv::kExpNan;
        float e1 = v_nan ? 0.f : (float)(vb - (kv::kExpBias + kRef));  // over kRef

        ok = ok && wait.warp(&sh.s_full, n & 1);
        ptx::tc_fence_after();
        uint64_t d2[RW / 2];  // scores in base 2 above the running maximum
        float high = -INFINITY;
        const uint64_t kf2 = ptx::pack2(kf, kf);
#pragma unroll
        for (int c = 0; c < RW; c += C::kStep) {
          if (c < used) {
            constexpr int K = C::kStep;
            uint32_t raw[NT * K];
#pragma unroll
            for (int q = 0; q < NT; ++q) tmem_ld<K>(col_s + q * RW + c, raw + q * K);
            wait_ld<NT * K>(raw);
            const uint64_t inv2 = ptx::pack2(1.f / kTerm, 1.f / kTerm);
#pragma unroll
            for (int r = 0; r < K; r += 4) {
              const ulonglong2 mul = *reinterpret_cast<const ulonglong2*>(&rw.mul[w * RW + c + r]);
              const ulonglong2 nm = *reinterpret_cast<const ulonglong2*>(&g.neg_m[c + r]);
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                auto pair = [&](int q) {
                  return ptx::pack2(__uint_as_float(raw[q * K + r + e]),
                                    __uint_as_float(raw[q * K + r + e + 1]));
                };
                uint64_t v = pair(NT - 1);
#pragma unroll
                for (int q = NT - 2; q >= 0; --q) v = ptx::ffma2(v, inv2, pair(q));
                d2[(c + r + e) / 2] =
                    ptx::ffma2(v, ptx::fmul2(kf2, e ? mul.y : mul.x), e ? nm.y : nm.x);
              }
            }
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sh.s_free);
        if (!plain) {
#pragma unroll
          for (int r = 0; r < RW; r += 2) {
            float d0, d1;
            ptx::unpack2(d2[r / 2], d0, d1);
            if (dead || key >= rw.lim[w * RW + r]) d0 = -INFINITY;
            if (dead || key >= rw.lim[w * RW + r + 1]) d1 = -INFINITY;
            d2[r / 2] = ptx::pack2(d0, d1);
          }
        }
#pragma unroll
        for (int r = 0; r < RW; r += 2) {
          if (r / C::kStep * C::kStep < used) {
            float d0, d1;
            ptx::unpack2(d2[r / 2], d0, d1);
            high = ptx::fmax3(high, d0, d1);
          }
        }

        // Does a row rise above its maximum by more than kRise? Then the
        // largest s + e of each row over the tile is its new one.
        const bool up = high + e1 > kRise;
        const bool rise = any_of(bare || up || !ok);
        // An exponent that the reference does not serve.
        if (!dead && fabsf(e1) > kWide) sh.again = 1;
        // P's buffer is free: the product that read it two tiles ago was
        // issued before these scores, whose completion covers it. With one
        // buffer the product of the tile before has to be waited for.
        if (C::kPBufs == 1 && n > 0) ok = ok && wait.warp(&sh.o_done[(n - 1) & 1], ((n - 1) >> 1) & 1);
        if (rise) {
          // A row of zeros has the exponent of 1 whatever its neighbours have. It
          // adds nothing under any exponent, and as one of 1 it would be the
          // maximum of keys whose values are small, whose terms then vanish.
          // Looked at only where it could set a maximum.
          bool zero = false;
          const bool look = (bare || up) && !dead && vb == kv::kExpBias;
          if (__any_sync(0xffffffffu, look)) {
            // (The products wait for the tile too, and report one that fails to come.)
            const int st = (2 * n + 1) % NS;
            if (wait_along(&sh.kv_full[st], ((2 * n + 1) / NS) & 1, &sh.abort) && look)
              zero = zero_row<D>(smem + st * C::kSlotBytes, tid);
          }
          // A maximum that zeros set all the same is kWide below their score. It is
          // right unless values are met below it: beside them in a first tile, in
          // the first tile with any behind tiles of zeros, or if it rises later.
          if (zero) e1 = bare && !first ? -INFINITY : -kWide;
          if (zero && !first && high - kWide > kRise) sh.again = 1;
          if (bare) {
            const bool solid = __any_sync(0xffffffffu, !dead && !zero && !v_nan);
            if (lane == 0) reinterpret_cast<uint8_t*>(&g.solid)[wq] = solid;
          }
          float top = -INFINITY;
#pragma unroll
          for (int r = 0; r < RW; r += 2) {
            if (r / C::kStep * C::kStep < used) {
              float d0, d1;
              ptx::unpack2(d2[r / 2], d0, d1);
              d0 = warp_max(d0 + e1);
              d1 = warp_max(d1 + e1);
              if (lane == r) top = d0;
              if (lane == r + 1) top = d1;
            }
          }
          if (lane < RW) reinterpret_cast<float*>(&g.top[lane])[wq] = top;
          if (any_of(!ok)) {
            left = true;
            break;
          }
          const bool solid = g.solid != 0;
          float f_lane = 1.f;
          if (lane < RW) {
            const float4 v4 = g.top[lane];
            const float v = fmaxf(fmaxf(v4.x, v4.y), fmaxf(v4.z, v4.w));
            if (bare && !first && v < -1.f && v > -INFINITY) sh.again = 1;
            float by = 0.f;
            if (v > (first ? -INFINITY : kRise)) {
              by = v;
              f_lane = first ? 0.f : ptx::ex2(-v);
              m_lane += v;
            }
            g.step[lane] = -by;
            g.neg_m[lane] = -m_lane;
          }
          __syncwarp();
#pragma unroll
          for (int r = 0; r < RW; r += 4) {
            if (r / C::kStep * C::kStep < used) {
              const ulonglong2 by = *reinterpret_cast<const ulonglong2*>(&g.step[r]);
              d2[r / 2] = ptx::fadd2(d2[r / 2], by.x);
              d2[r / 2 + 1] = ptx::fadd2(d2[r / 2 + 1], by.y);
            }
          }
          if (first && solid && __any_sync(0xffffffffu, zero)) {
            float above = -INFINITY;
#pragma unroll
            for (int r = 0; r < RW; r += 2) {
              if (r / C::kStep * C::kStep < used) {
                float d0, d1;
                ptx::unpack2(d2[r / 2], d0, d1);
                above = ptx::fmax3(above, d0, d1);
              }
            }
            if (zero && above > kWide - 1.f) sh.again = 1;
          }
          bare = !solid;
          if (t > s.t0) {
            // The sums so far, rescaled; O when the tile before is in it.
            const uint32_t rose = __ballot_sync(0xffffffffu, f_lane != 1.f);
            ok = ok && wait.warp(&sh.o_done[(n - 1) & 1], ((n - 1) >> 1) & 1);
            ptx::tc_fence_after();
#pragma unroll
            for (int c = 0; c < RW; c += 8) {
              if ((rose >> c) & 0xffu) {
                uint32_t o8[NT * 8];
#pragma unroll
                for (int q = 0; q < NT; ++q) tmem_ld<8>(col_o + q * RW + c, o8 + q * 8);
                wait_ld<NT * 8>(o8);
#pragma unroll
                for (int r = 0; r < 8; r += 2) {
                  const float f0 = __shfl_sync(0xffffffffu, f_lane, c + r);
                  const float f1 = __shfl_sync(0xffffffffu, f_lane, c + r + 1);
                  l2[(c + r) / 2] = ptx::fmul2(l2[(c + r) / 2], ptx::pack2(f0, f1));
#pragma unroll
                  for (int q = 0; q < NT; ++q) {
                    o8[q * 8 + r] = __float_as_uint(__uint_as_float(o8[q * 8 + r]) * f0);
                    o8[q * 8 + r + 1] = __float_as_uint(__uint_as_float(o8[q * 8 + r + 1]) * f1);
                  }
                }
#pragma unroll
                for (int q = 0; q < NT; ++q) tmem_st8(col_o + q * RW + c, o8 + q * 8);
              }
            }
            ptx::tmem_wait_st();
          }
        }
        // p, its sum, and the key's row of P: the terms side by side. A key
        // that some rows do not see may have a NaN factor: their product with
        // it is then not formed (kPick). The factor, 8 * 2^e over the reference,
        // is a power of two by its bits (of exponents near the reference; shares
        // with others are computed again).
        const float vf = dead ? 0.f : __int_as_float((vb + (kPShift - kRef)) << 23);
        uint8_t* const p_tile = p_tiles + n % C::kPBufs * C::kPBytes;
        auto emit = [&](auto pick) {
          constexpr bool kPick = decltype(pick)::value;
          const float f = kPick && v_nan ? __int_as_float(0x7fc00000) : vf;
          const uint64_t vf2 = ptx::pack2(f, f);
#pragma unroll
          for (int c = 0; c < RW; c += 8) {
            if (c < used) {
              uint32_t y[4];
#pragma unroll
              for (int r = 0; r < 8; r += 2) {
                float d0, d1, y0, y1;
                ptx::unpack2(d2[(c + r) / 2], d0, d1);
                const uint64_t p = ptx::pack2(ptx::ex2(d0), ptx::ex2(d1));
                l2[(c + r) / 2] = ptx::fadd2(l2[(c + r) / 2], p);
                ptx::unpack2(ptx::fmul2(p, vf2), y0, y1);
                if (kPick && d0 == -INFINITY) y0 = 0.f;
                if (kPick && d1 == -INFINITY) y1 = 0.f;
                y[r / 2] = h2(y0, y1);
              }
              uint2 t8[NT];
              terms8<NT>(y[0], y[1], y[2], y[3], t8);
#pragma unroll
              for (int q = 0; q < NT; ++q)
              {
                const int col = w * C::kN + q * RW + c;
                *reinterpret_cast<uint2*>(p_tile + col / C::kPitch * (kTileKeys * C::kPitch) +
                                          swz<C::kPitch>(tid, col % C::kPitch)) = t8[q];
              }
            }
          }
        };
        if (__any_sync(0xffffffffu, v_nan))
          emit(std::true_type());
        else
          emit(std::false_type());
        // Rows of V that are not this item's keys (the end of a page, a page
        // not brought in) may hold anything, NaN codes among them: zeros.
        if (w == 0 && first_key + kTileKeys > s.len) {
          const int st = (2 * n + 1) % NS;
          ok = ok && wait.warp(&sh.kv_full[st], ((2 * n + 1) / NS) & 1);
          if (dead) {
            uint4* row = reinterpret_cast<uint4*>(smem + st * C::kSlotBytes + tid * D);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) row[c] = make_uint4(0, 0, 0, 0);
          }
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sh.p_full[n & 1]);
      }
      if (left) break;

      // ------------------------------------------------------ the item's result
      {
        float l[RW];
#pragma unroll
        for (int r = 0; r < RW; r += 2) ptx::unpack2(l2[r / 2], l[r], l[r + 1]);
        const float v = warp_sums<RW>(l);
        constexpr int kEach = 32 / RW;  // lanes that hold the same row's sum
        if (lane % kEach == 0) reinterpret_cast<float*>(&g.sum[lane / kEach])[wq] = v;
      }
      if (any_of(!ok)) break;
      const bool whole = s.t0 == 0 && s.t1 == s.nt;
      const int part = 2 * cta + (k > 0 ? 1 : 0);
      // Lane r looks after row r (its maximum is there).
      float inv_lane = 0.f;
      int id_lane = -1;
      if (lane < used) {
        id_lane = rw.row_id[w * RW + lane];
        const float sum = sum_of(g.sum[lane]);
        const float top = sum == 0.f ? -INFINITY : m_lane;
        // 2^kRef / 8, what P was taken over, by the sum
        inv_lane = sum == 0.f ? 0.f : __fdividef(__int_as_float((127 + kRef - kPShift) << 23), sum);
        if (wq == 0) {
          if (!whole)
            a.part_ml[(long long)part * C::kRows + w * RW + lane] = make_float2(top, sum);
          else if (!a.own_rows)
            a.full_ml[id_lane] = make_float2(top, sum);
          else if (a.lse)
            a.lse[id_lane] = sum == 0.f ? -INFINITY : ln_of(top, sum);
        }
      }
      // (Should this wait give up, the next barrier ends the block.)
      ok = ok && wait.warp(&sh.o_done[(n - 1) & 1], ((n - 1) >> 1) & 1);
      ptx::tc_fence_after();
      // O^T: a thread has one d of every row; with D = 64 the upper half of the
      // lanes repeats the lower and takes the odd rows.
      const int d = tid % D;
#pragma unroll
      for (int c = 0; c < RW; c += 8) {
        if (c < used) {
          uint32_t raw[NT * 8];
#pragma unroll
          for (int q = 0; q < NT; ++q) tmem_ld<8>(col_o + q * RW + c, raw + q * 8);
          wait_ld<NT * 8>(raw);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int r = c + e;
            const float inv = __shfl_sync(0xffffffffu, inv_lane, r);
            const long long to =
                whole ? rw.off[w * RW + r] : ((long long)part * C::kRows + w * RW + r) * D;
            float v = __uint_as_float(raw[(NT - 1) * 8 + e]);
#pragma unroll
            for (int q = NT - 2; q >= 0; --q)
              v = fmaf(v, 1.f / kTerm, __uint_as_float(raw[q * 8 + e]));
            v *= inv;
            if (r < used && (D == 128 || (r & 1) == tid / 64)) {
              if (!whole)
                a.part_o[to + d] = v;
              else if (!a.own_rows)
                a.full_o[to + d] = v;
              else if (kBf16)
                reinterpret_cast<__nv_bfloat16*>(a.o)[to + d] = __float2bfloat16(v);
              else
                reinterpret_cast<__half*>(a.o)[to + d] = __float2half(v);
            }
          }
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sh.q_free[k & 1]);
      if (C::kHelperQ ? last : !walk.next(a, C::kItemCost, s)) break;
    }
    end_sync();  // nothing is under way any more: the ring is free
    if (sh.again && !sh.abort) share_again<C, kBf16>(a, sh.start, reinterpret_cast<float*>(smem));
  }

  if (warp == C::kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(sh.tmem, C::kTmemCols);
  }
  // A launch that overlaps the one before it ends after it: whoever waits for
  // this one has both.
  if (a.early) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// --------------------------------------------------------------------- joining
// Sum of parts of one row, spread over a warp: lane holds D / 32 values. A part
// is its result o, the maximum m that its weights are relative to and their sum
// l = 2^k x; it weighs 2^m l, and the joined row's m is the largest m + k. Results
// are at most as large as values are: kLess keeps the sum of up to a thousand of
// them, each weighing less than 2, inside fp32.
template <int D>
struct RowSum {
  static constexpr int V = D / 32;
  static constexpr float kLess = 1.f / 2048;
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
      const int k = log2_below(ml.y);
      const float lead = ml.x + (float)k;
      const float top = fmaxf(m, warp_max(lead));
      const float use = top == -INFINITY ? 0.f : top;
      const float keep = ptx::ex2(m - use);
      float w = ptx::ex2(lead - use) * over_log2(ml.y, k), sum = w;
      w *= kLess;
#pragma unroll
      for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
      l = l * keep + sum;
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] *= keep;
      m = top;
      // The rows come in sixteens that are all on their way at once; behind
      // the last one it is read again, with no weight.
      constexpr int kFly = 16;
#pragma unroll 1
      for (int i = 0; i < here; i += kFly) {
        float x[kFly][V];
#pragma unroll
        for (int u = 0; u < kFly; ++u) load(po + at(i0 + min(i + u, here - 1)) * D + lane * V, x[u]);
#pragma unroll
        for (int u = 0; u < kFly; ++u) {
          const float wi = __shfl_sync(0xffffffffu, w, min(i + u, here - 1));
#pragma unroll
          for (int e = 0; e < V; ++e) o[e] = fmaf(i + u < here ? wi : 0.f, x[u][e], o[e]);
        }
      }
    }
  }
  template <bool kBf16>
  __device__ __forceinline__ void store(const Args& a, int b, int h, int i) const {
    const int lane = threadIdx.x % 32;
    const float inv = l == 0.f ? 0.f : 1.f / (kLess * l);
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
          l == 0.f ? -INFINITY : ln_of(m, l);
  }
};

// Joins the parts of the item that block `blockIdx.x` of the first kernel
// began and did not end; a warp per row. The bound of four blocks an SM lets
// the compiler hold a batch of rows in registers: without it it took 32 and
// waited for each row by itself (75 parts: 13 us).
template <int D, bool kBf16>
__global__ void __launch_bounds__(128, 4) decode_join_kernel(const Args a, int tile_rows) {
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
  int row_tiles, tile_rows, grid;
};

// Joins every row's prefix with what is behind it; a warp per row.
template <int D, bool kBf16>
__global__ void __launch_bounds__(128, 4) prefix_join_kernel(const Args a, const Set pre, const Set own) {
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
    } else if (it.w == kItemParts && it.x >= 0 && it.x <= it.y && it.y < s.grid && it.z >= 0 &&
               it.z < 2 * s.grid) {
      // (A block that gave up waiting has not said where its later items are:
      // the workspace holds anything there.)
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
  // The units of work number less than 2^31, whatever the lengths are.
  const int64_t group = p->heads / p->cache.heads_kv;
  const int64_t tiles =
      (p->cache.max_pages * p->cache.page_size + 2 * kTileKeys - 1) / kTileKeys + kMostItemCost;
  for (int64_t rows : {p->seqlen_q * group, p->seqlen_q * group * p->cache.batch}) {
    const int64_t seqs = rows == p->seqlen_q * group ? p->cache.batch : 1;
    if (seqs * p->cache.heads_kv * ((rows + 7) / 8) > (1ll << 31) / tiles - 1)
      return fa8_note_error(FA8_ERR_UNSUPPORTED, "fa8_decode: too many key tiles for one call");
  }
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
  if (rows <= 32) return {16, 2};
  return {16, 4};
}
constexpr int kSmCount = 148;

// Workspace of one set of items.
struct Layout {
  Shape shape;
  int64_t row_tiles, items, grid;
  int64_t part_o, part_ml, seg, item, full_o, full_ml, end;  // byte offsets
};
int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

// Keys that are taken from row 0 of the table for all sequences: those in whole
// pages of the prefix, however they are met.
int64_t shared_len(const fa8_decode_params* p) {
  return p->prefix_len / p->cache.page_size * p->cache.page_size;
}

// Whether a prefix has a set of items of its own. Three launches in a row take
// 16 us however little there is to do, two 10; met by every sequence for
// itself (from the same pages, in L2) the prefix is more tiles to each block.
// Together / one by one, us, 32 heads on 8, D = 128, 296 blocks: 16 sequences
// behind 1024 (3.5 tiles a block) 24 / 17, behind 2048 (7) 26 / 21, 32 behind
// 2048 (14) 29 / 31, 64 behind 2048 (28) 40 / 51; 16 heads of D = 64, 444
// blocks: 8 behind 1000 (2.3) 21 / 15, 48 behind 1024 (14) 30 / 39.
bool prefix_apart(const fa8_decode_params* p) {
  const int64_t rows = p->seqlen_q * (p->heads / p->cache.heads_kv);
  const Shape s = shape_for(rows);
  const int64_t tiles = (rows + s.tile_rows() - 1) / s.tile_rows() * p->cache.batch *
                        p->cache.heads_kv * ((shared_len(p) + kTileKeys - 1) / kTileKeys);
  return tiles > 10 * kSmCount * resident((int)p->cache.head_dim, s.rw, s.nwg);
}

Layout layout_of(const fa8_decode_params* p, bool prefix_set, int64_t at) {
  Layout l;
  const int64_t D = p->cache.head_dim, B = p->cache.batch;
  const int64_t rows = p->seqlen_q * (p->heads / p->cache.heads_kv) * (prefix_set ? B : 1);
  l.shape = shape_for(rows);
  l.row_tiles = (rows + l.shape.tile_rows() - 1) / l.shape.tile_rows();
  l.items = p->cache.heads_kv * l.row_tiles * (prefix_set ? 1 : B);
  l.grid = (int64_t)kSmCount * resident((int)D, l.shape.rw, l.shape.nwg);
  const int64_t parts = 2 * l.grid * l.shape.tile_rows();
  const bool two = prefix_apart(p);
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
  static int regs[64];
  if (dev < 0 || dev >= 64) return fa8_note_error(FA8_ERR_INVALID_ARG, "device index out of range");
  auto kernel = decode_kernel<C, kBf16>;
  std::call_once(flags[dev], [&] {
    errs[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    cudaFuncAttributes at;
    if (errs[dev] == cudaSuccess) errs[dev] = cudaFuncGetAttributes(&at, kernel);
    if (errs[dev] == cudaSuccess) regs[dev] = at.numRegs;
  });
  if (errs[dev] != cudaSuccess) return fa8_note_cuda_error(errs[dev], "decode kernel attributes");
  // The register split draws on what the block is launched with: with less than
  // its sum a warpgroup would wait for registers for ever. (The build checks it.)
  if (C::NWG * C::kRegsSoft + C::kRegsHelp > (C::NWG + 1) * regs[dev]) {
    char msg[160];
    snprintf(msg, sizeof(msg),
             "fa8_decode: this build's kernel has %d registers a thread, its split between the "
             "warps needs %d: rebuild with the compiler and flags of _build.py",
             regs[dev], C::kRegsLaunch);
    return fa8_note_error(FA8_ERR_UNSUPPORTED, msg);
  }
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
  a.by_row_tiles = Divisor::of(a.row_tiles);
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
  if (l.shape.nwg == 4) return launch_set<Cfg<D, NT, 16, 4>, kBf16>(a, tk, tv, grid, dev, stream);
  if (l.shape.nwg == 2) return launch_set<Cfg<D, NT, 16, 2>, kBf16>(a, tk, tv, grid, dev, stream);
  if (l.shape.rw == 16) return launch_set<Cfg<D, NT, 16, 1>, kBf16>(a, tk, tv, grid, dev, stream);
  return launch_set<Cfg<D, NT, 8, 1>, kBf16>(a, tk, tv, grid, dev, stream);
}

template <int D, bool kBf16>
int run(const fa8_decode_params* p, Args a, char* ws, int dev, cudaStream_t stream) {
  cudaError_t e;
  if (!prefix_apart(p)) {
    const Layout l = layout_of(p, false, 0);
    a.own_rows = 1;
    a.shared_pages = (int)(p->prefix_len / p->cache.page_size);
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
    b.prefix_len = (int)shared_len(p);
    int st = run_set<D, kBf16>(p, b, l0, ws, dev, stream);
    if (st) return st;
    b = a;
    b.key0 = (int)shared_len(p);
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
      s.grid = (int)l.grid;
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
      p->cache.page_size <= 0 || p->prefix_len > p->cache.max_pages * p->cache.page_size ||
      p->heads % p->cache.heads_kv != 0) {
    fa8_note_error(FA8_ERR_INVALID_ARG, "fa8_decode_workspace_size: sizes that fa8_decode refuses");
    return -1;
  }
  if (p->cache.batch == 0 || p->heads == 0 || p->seqlen_q == 0) return 0;
  if (!prefix_apart(p)) return layout_of(p, false, 0).end;
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
  const int page = (int)p->cache.page_size;
  a.box = std::min(page, kTileKeys);
  a.by_page = Divisor::of(page);
  a.by_group = Divisor::of(a.group);
  a.by_seq_rows = Divisor::of(a.group * a.seqlen_q);
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
