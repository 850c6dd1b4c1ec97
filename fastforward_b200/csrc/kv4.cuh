// The 4-bit paged K/V cache: record layout, sequence bookkeeping and nibble arithmetic
// shared by its writer, its reader and the attention kernels.
//
// A page holds 64 tokens.  Per (page, K/V head) one record of 9216 contiguous bytes, so one
// bulk copy brings everything a tile of 64 keys needs:
//   [0, 4096)     K codes, 64 bytes a token.  Byte 16 t + 4 j + e / 2, nibble e % 2 holds
//                 channel 32 j + 8 t + e (t, j in 0..3, e in 0..7): 16 bytes hold, for each
//                 scale group j, the eight channels that one lane of an MMA fragment needs.
//   [4096, 8192)  V codes, 64 bytes a token: eight chunks of 8 bytes, chunk g at position
//                 g ^ (token & 4); its nibble i holds channel 8 i + g.  The exchange of the
//                 two halves for tokens 4..7 of eight spreads the fragment loads over all
//                 shared-memory banks.
//   [8192, 8704)  K scales bf16 [64][4];  [8704, 9216)  V scales bf16 [64][4].
// A group of 32 channels has the scale s = the smallest number of five significant bits that
// is >= max|x| / 7, codes q = rint(x / s) in -7..7, nibble q + 8.  Five bits times three fit
// bf16's eight, so every held value q s is exact in bf16 and any kernel may multiply codes
// and scales before or after its products with the same result.  The rounding up of s costs
// at most 1/16 of a step and never clips.  max|x| < 2^-100 gives s = 0; a group with a
// non-finite value (or one of 2^127 and more) gives s = NaN, so the row reads as NaN.
#pragma once
#include "common.cuh"

namespace kv4 {

constexpr int D = 128;
constexpr int PAGE = FFB_KV4_PAGE;
constexpr int RECORD = FFB_KV4_RECORD;
constexpr int V_CODES = 4096, K_SCALES = 8192, V_SCALES = 8704;
static_assert(PAGE == 64 && RECORD == 9216, "record layout");

// What every entry is told about the cache and the rows of the call.
struct Seqs {
  uint8_t* pages;        // [num_pages][HK][RECORD]
  const int* table;      // [B] rows of max_pages page ids, table_stride apart
  const int* row_start;  // [B + 1]: rows [row_start[b], row_start[b + 1]) of the call are sequence b's newest
  const int* ctx_len;    // [B]: tokens of sequence b with those rows
  int num_pages, max_pages, B, T, HK;
  int64_t table_stride;
};

// The sequence that row t belongs to, or -1 (rows before the first or behind the last).
__device__ __forceinline__ int seq_of(const Seqs& s, int t) {
  if (t < __ldg(s.row_start) || t >= __ldg(s.row_start + s.B)) return -1;
  int lo = 0, hi = s.B;  // the first b with row_start[b + 1] > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(s.row_start + mid + 1) > t) hi = mid;
    else lo = mid + 1;
  }
  return lo < s.B ? lo : -1;
}

// The record of (sequence b, position pos, head h), or NULL when the position is outside the
// table or the page id outside the cache.
__device__ __forceinline__ uint8_t* record_of(const Seqs& s, int b, int64_t pos, int h) {
  if (pos < 0 || pos >= (int64_t)s.max_pages * PAGE) return nullptr;
  const int page = __ldg(s.table + b * s.table_stride + pos / PAGE);
  if (page < 0 || page >= s.num_pages) return nullptr;
  return s.pages + ((int64_t)page * s.HK + h) * RECORD;
}

// Arguments of the attention kernels.
struct AttnArgs {
  const uint16_t* q;  // [HQ, T, 128]
  uint16_t* out;      // [T, HQ, 128]
  uint64_t* flags;    // [CTAs][2]: `tag` once that part is written (register path, equal runs); behind them a failed run's mark
  uint64_t tag;
  float* part_o;      // partial rows of 128, relative to their maxima: register path [CTAs][2][columns], TC [cut][splits][256]
  float* part_ml;     // their (maximum, sum) pairs
  Seqs seqs;
  int HQ, splits, window, sinks;
  int whole, cut;  // TC: items that one CTA does, and before them those in `splits` shares
  float scale_log2;
  uint32_t* errors;  // TC: the device's error word
};

// The TC path's items: 256 columns ((row, head of the group) pairs) of a K/V head of a sequence,
// numbered sequence by sequence, tile by tile, the heads of a tile next to each other.  Found by a
// converged warp, 32 sequences a step; r0 = -1 behind the last item.
struct TcItem {
  int b, kvh, tile, r0, rows, ctx;
};
__device__ __forceinline__ TcItem tc_item(const AttnArgs& a, int item) {
  const Seqs& sv = a.seqs;
  const int lane = threadIdx.x & 31, G = a.HQ / sv.HK, kvh = item % sv.HK;
  int t = item / sv.HK;
  for (int b0 = 0; b0 < sv.B; b0 += 32) {
    const int b = b0 + lane;
    int r0 = 0, rows = 0, ctx = 0;
    if (b < sv.B) {
      ctx = max(__ldg(sv.ctx_len + b), 0);
      r0 = min(max(__ldg(sv.row_start + b), 0), sv.T);
      rows = min(max(__ldg(sv.row_start + b + 1), r0), sv.T) - r0;
    }
    const int tiles = (rows * G + 255) >> 8;
    int sum = tiles;  // of the lanes up to this one
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += other;
    }
    const uint32_t in = __ballot_sync(0xffffffffu, sum > t);
    if (in) {
      const int src = __ffs(in) - 1;
      return {b0 + src, kvh, __shfl_sync(0xffffffffu, t - sum + tiles, src), __shfl_sync(0xffffffffu, r0, src),
              __shfl_sync(0xffffffffu, rows, src), __shfl_sync(0xffffffffu, ctx, src)};
    }
    t -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return {0, 0, 0, -1, 0, 0};
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What a row's scores are multiplied with when its maximum (base 2) is m.  Up to 2^30 in size nothing: 1.
// Beyond, fp32 scores next to each other are 32 and more apart, so that only their order counts, but
// x mul - m in one rounding may be off by as much as m is, by far more than exp2 holds: a power of two
// brings m between 2^29 and 2^30, where it is off by 32 at most.
__device__ __forceinline__ float vast_scale(float m) {
  const uint32_t e = (__float_as_uint(m) >> 23) & 255u;
  return e < 127 + 30 ? 1.f : __uint_as_float((127 + 29 + 127 - e) << 23);
}
// Nibbles i and i + 4 of w as the bf16 pair (136 + code).
__device__ __forceinline__ uint32_t pair136(uint32_t w, int i) { return ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u; }
__device__ __forceinline__ uint32_t minus136(uint32_t w) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&w), __floats2bfloat162_rn(136.f, 136.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// mbar_wait_bounded for waits that are expected to take long: the hardware may hold the thread for up
// to 10 us a try, so that waiting warps leave the issue slots to the others.
__device__ __forceinline__ bool wait_held(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  for (uint32_t i = 0; i < (1u << 24); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(10000u)
        : "memory");
    if (ok) return true;
    if (*abort || global_timer_ns() - t0 > 2000000000ull) return false;
  }
  return false;
}
// The pages that a tile of rows [first, last] (positions) reads: the first n_sink pages, then
// [first_page, first_page + n - n_sink).
struct PageSet {
  int n, n_sink, first_page, first_key, kend;
};
__device__ __forceinline__ PageSet pages_of(int pos_lo, int pos_hi, int max_pages, int window, int sinks) {
  PageSet s;
  s.kend = min(pos_hi + 1, max_pages * PAGE);
  s.first_key = window > 0 ? max(0, pos_lo - window + 1) : 0;
  s.first_page = s.first_key / PAGE;
  s.n_sink = window > 0 ? min((min(sinks, max(s.kend, 0)) + PAGE - 1) / PAGE, s.first_page) : 0;
  s.n = s.kend > 0 ? s.n_sink + max(0, (s.kend + PAGE - 1) / PAGE - s.first_page) : 0;
  return s;
}

}  // namespace kv4

namespace ffb {
// Whether n bytes at a and m bytes at b share any (host).
inline bool overlap(const void* a, int64_t n, const void* b, int64_t m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + (uint64_t)m && y < x + (uint64_t)n;
}
// The argument checks that every kv4 entry shares (host): FFB_OK or FFB_EINVAL with a message.
int kv4_check(const char* who, const void* pages, const int* table, const int* row_start, const int* ctx_len,
              int num_pages, int64_t table_stride, int max_pages, int B, int T, int HK);
}  // namespace ffb
