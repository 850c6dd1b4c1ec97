// Attention over the 4-bit paged K/V cache (layout: kv4.cuh) for few query rows a sequence:
// single-token decoding and short runs of new tokens.
//
//   o[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - m),  x_j = scale log2(e) q.k_j
// over the keys j <= the row's position, inside the window or among the first `sinks`.
//
// The floor is the bytes of the visible pages (144 a token and K/V head), so the kernel is
// built to keep bulk copies in flight and to spend few instructions a byte:
//   - an item is one (sequence, K/V head, 8 NT query columns); the columns are the (row, head of
//     the group) pairs, so a page is read once for all the query heads that share it.  A CTA has
//     eight warps; two of them take a page, 32 tokens each, and every warp has a ring of its own of
//     STAGES such halves, filled by cp.async.bulk: no warp waits for another inside a share, and
//     page ids are read 32 at a time, so no load waits for one;
//   - the CTAs share out the pages of all items in equal runs, whatever the lengths of the
//     sequences (they are on the device, so every CTA sums them up itself), or, where these are even
//     enough, take an item each; an item cut by a run's
//     end leaves fp32 partials, which the CTA that has its last page adds up at the end of its own
//     run (it waits only for CTAs before it; a second launch cost 6 us).  With few pages an item
//     (WHOLE) each item is one CTA's.  The first pages and the queries of a CTA's next item are on
//     their way while it works on this one;
//   - the products run on mma.sync m16n8k16 with the tokens on M and the query columns on N
//     (S^T = K Q^T, O^T = V^T P^T): with G <= 8 heads a group a tcgen05 tile of 128 rows
//     would be nearly empty, and its operands would have to be written to shared memory as
//     bf16, four times the bytes of the codes.  Here a code becomes an operand in a register;
//   - every fragment is a chain of dependent instructions, mostly on the half-rate logic pipe, and an SM
//     has 16 warps to overlap them, so the nibbles are used where they lie.  Masked with 0x000F / 0x00F0
//     a pair of them is a pair of fp16 (K) or bf16 (V) subnormals, u 2^-24 and 16 u 2^-24 or u 2^-133 and
//     16 u 2^-133 (u = code + 8; eight bits are linear across bf16's first two binades), which the tensor
//     core multiplies exactly.  Two masks, a shift by 8 and two masks more make eight operands;
//   - K: Q is scaled by a power of two per column into fp16's upper range (its eight bits stay
//     exact down to 2^-28 of the column's largest value), a sixteenth of it for the channels in
//     the upper nibbles.  A group's scale multiplies its fp32 sum; what u is too large by,
//     sum_group 8 s_group sum(q), is one more MMA of the scales themselves with 8 sum(q) in three
//     bf16 parts, which the scores start from;
//   - V: probabilities are held 2^64 times too large (so that products with the subnormals are
//     normal numbers; |v| must stay below 2^57, and a sum, held 2^-69 too small, is exact to 2^-80: bf16's
//     bits down to about 2^-68), V's scale multiplies one before its only rounding
//     to bf16, once per group of channels; movmatrix turns the scores' layout into that of the
//     second product's operand.  A second MMA with the constants -8 2^-133 and -128 2^-133 takes
//     the 8 off (half the tensor work, but no instruction a code);
//   - the running maximum moves only when a score passes it by more than 8 (in base 2), which
//     a vote finds: p <= 2^8, nothing overflows, and the rescaling is rare.
// S, the maxima, the sums and O are fp32; P (times V's scale) is rounded to bf16, the type of
// the tensor core's operand, with relative error 2^-8 of each term.
// Measured (32 + 8 heads unless said): 64 sequences of 777 to 8192 tokens 90 us, 3.3 TB/s; one of
// 131001 tokens 48.5 us, 3.1 TB/s; 16 of 3333 and 4096 tokens, 64 + 8 heads, 31.5 us, 2.2 TB/s; 16 with a
// window of 4096 33 us, 2.3 TB/s; one of 321 tokens 8.2 us, latency.  About 350 instructions a fragment of 16
// tokens.  No pipe is full (issue slots 52%, logic pipe 51% of active cycles): warps wait for their own
// last instruction, and at the barriers where an item ends (about 5 us a change); the copies alone would
// run at 6 TB/s.
#include "kv4.cuh"
#include "pdl.cuh"

#include <cuda_fp16.h>
#include <math.h>

#include <atomic>
#include <chrono>

namespace {

using namespace kv4;

constexpr int WARPS = 8;
constexpr int THREADS = 32 * WARPS;
constexpr int GROUPS = WARPS / 2;     // pages that a CTA has in hand at once
constexpr int HALF = PAGE / 2;        // tokens of a page that a warp takes
// A half page in shared memory: K codes, V codes, K scales, V scales.
constexpr int HALF_CODES = HALF * 64, HALF_SCALES = HALF * 8;
constexpr int HALF_V = HALF_CODES, HALF_KS = 2 * HALF_CODES, HALF_VS = HALF_KS + HALF_SCALES;
constexpr int HALF_BYTES = HALF_VS + HALF_SCALES;
constexpr int QROW = 2 * D + 16;      // byte pitch of a query row (spreads the banks)
constexpr int CS = D + 4;             // fp32 pitch of a column in the final exchange (spreads the banks)
constexpr float LAZY = 8.f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float UNSEEN = 3e38f;       // 64 - maximum before the first score: finite, so that -inf gives exp2(-inf)

constexpr int MIN_PAGES = GROUPS;     // fewest pages worth a CTA: one a group
constexpr int ITEM_PAGES = 8;         // what starting and ending an item takes, in pages
// Items are not cut where the longest has at most so many pages more than an equal run: us apart / cut,
// 32 + 8 heads, in a table of 128 pages: 32 sequences of 256 tokens 11.0 / 17.8, of 2048 tokens 28.3 / 34.1
// (5 pages more); 8 of 640 tokens (14 more) 13.7 / 13.7.
constexpr int APART = 10;

// Sequence b's rows, pages and items in the run of pages that the CTAs share: its items, HK for
// each tile of `qt` columns, one after the other, each with ITEM_PAGES for its start and end and
// the pages that any of its rows sees.
struct Seq {
  int r0, S, ctx, tiles;
  PageSet ps;
  __device__ __forceinline__ int pages() const { return max(ps.n, 1); }  // an item of no pages still writes its zeros
  __device__ __forceinline__ int64_t weight(int HK) const { return (int64_t)tiles * HK * (ITEM_PAGES + pages()); }
};
__device__ __forceinline__ Seq seq_at(const AttnArgs& a, int b, int qt) {
  const Seqs& s = a.seqs;
  Seq q;
  q.r0 = min(max(__ldg(s.row_start + b), 0), s.T);
  q.S = min(max(__ldg(s.row_start + b + 1), q.r0), s.T) - q.r0;
  q.ctx = max(__ldg(s.ctx_len + b), 0);
  q.tiles = (q.S * (a.HQ / s.HK) + qt - 1) / qt;
  q.ps = pages_of(q.ctx - q.S, q.ctx - 1, s.max_pages, a.window, a.sinks);
  return q;
}
// The first sequence after b, which has no rows, that has some; B if there is none.  Row starts ascend, so a
// thousand empty sequences cost a few loads (one after the other they took 150 us).
__device__ __forceinline__ int next_with_rows(const Seqs& s, int b) {
  const int end = __ldg(s.row_start + b + 1);
  int step = 1;
  while (b + step < s.B && __ldg(s.row_start + b + step + 1) <= end) {
    b += step;
    step *= 2;
  }
  int lo = b, hi = min(b + step, s.B);  // lo has no rows, hi has or is B
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(s.row_start + mid + 1) <= end) lo = mid;
    else hi = mid;
  }
  return hi;
}
// One item's share, in shared memory: pages [i0, i1) of sequence b's list `ps` for one K/V head and
// the columns [c0, clast]; what every warp needs to know about it, found once by one thread.
struct Share {
  int b, kvh, c0, clast, i0, i1;
  int r0, pos0;            // the sequence's first row and its position
  int pos_lo, whole_lo, whole_hi;  // of the first column; page indexes [whole_lo, whole_hi) are seen in full by every column
  int entire;              // the whole item
  PageSet ps;
};
// Where a CTA stands in its run (moved on by one thread): what is left of it, the page `from` (from
// -ITEM_PAGES on) of item `item` of sequence b, that sequence; whether there is another share; the
// shares of this turn and the next; the first share, if it ends an item that began in another CTA.
struct Run {
  int64_t left;
  int b, item, from, more, items, known, failed;
  Seq seq;
  Share share[2], cut;
};

template <int NT>
struct Shape {
  // two CTAs an SM, so that one starts or ends while the other streams; 16 columns need the
  // registers (64 sums a thread) and the shared memory of one
  static constexpr int PER_SM = NT == 1 ? 2 : 1;
  static constexpr int STAGES = NT == 1 ? 2 : 4;  // half pages in a warp's ring
  static constexpr int RING = WARPS * STAGES * HALF_BYTES;
  static constexpr int EXCHANGE = WARPS * (2 * 8 * NT + 8 * CS) * 4;
  static constexpr int BARS = WARPS * STAGES * 8 + WARPS * 16 + sizeof(Run) + 16;
  // ring | exchange | Q fragments [NT][4][32] uint4 | query rows [8 NT][QROW], of this and the next item |
  // sums of 8 q [8 NT][4] | column factors, positions | barriers, schedule
  static constexpr int SMEM = RING + EXCHANGE + NT * 4 * 512 + 2 * 8 * NT * QROW + NT * 128 + NT * 64 + BARS + 128;
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// fp16 operands, the sum starting at zero.
__device__ __forceinline__ void mma16816_h0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma16816_h(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                           uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// bf16 operands, the sum starting at zero.
__device__ __forceinline__ void mma16816_0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                           uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// (x a, y b) in one instruction.
__device__ __forceinline__ float2 mul_pair(float x, float y, float a, float b) {
  float2 r;
  asm("{\n\t.reg .b64 v, w;\n\t"
      "mov.b64 v, {%2, %3};\n\tmov.b64 w, {%4, %5};\n\t"
      "mul.rn.f32x2 v, v, w;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x), "f"(y), "f"(a), "f"(b));
  return r;
}
// Part `i` (0, 1, 2) of v as a sum of three bf16 numbers.
__device__ __forceinline__ float bf16_part(float v, int i) {
  const float hi = round_bf(v), mid = round_bf(v - hi);
  return i == 0 ? hi : i == 1 ? mid : v - hi - mid;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// 16 bytes global -> shared, or zeros.
__device__ __forceinline__ void copy16(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void st_release_gpu_u64(uint64_t* p, uint64_t v) {
  asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
// mbarrier and bulk copy on shared-memory addresses held as integers.
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool arrived(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// The token of fragment row r (0..7): 2 <-> 3 and 6 <-> 7 trade places, so that the eight lanes
// of a load phase meet rows of both parities and, with V's exchanged halves, all banks.
__device__ __forceinline__ int token_of(int r) { return r ^ ((r >> 1) & 1); }

// A row's sums (maximum, sum of probabilities, four channels of O), and another part of the row added.
struct Sum {
  float top, l;
  float4 o;
};
__device__ __forceinline__ void add_part(Sum& s, float m, float l, float4 v) {
  if (m == -INFINITY && l == 0.f) return;  // nothing seen there
  const float top = fmaxf(s.top, m), fs = s.top == top ? 1.f : ex2(s.top - top), f = ex2(m - top);
  s.top = top;
  s.l = fmaf(l, f, s.l * fs);
  s.o.x = fmaf(v.x, f, s.o.x * fs);
  s.o.y = fmaf(v.y, f, s.o.y * fs);
  s.o.z = fmaf(v.z, f, s.o.z * fs);
  s.o.w = fmaf(v.w, f, s.o.w * fs);
}
__device__ __forceinline__ void store_row(uint16_t* out, const Sum& s, int lane) {
  const float r = s.l == 0.f ? 0.f : 1.f / s.l;
  *reinterpret_cast<uint2*>(out + 4 * lane) = make_uint2(pack_bf16(s.o.x * r, s.o.y * r), pack_bf16(s.o.z * r, s.o.w * r));
}

// What a call whose wait gave up leaves behind the flags (tags are odd: none is another call's).
__device__ __forceinline__ uint64_t failed_tag(uint64_t tag) { return tag ^ 1u; }
// a b / c, in 32 bits where that is enough (a 64-bit division takes hundreds of cycles).
__device__ __forceinline__ int64_t mul_div(int a, int64_t b, int c) {
  if (b < (1 << 22) && a < 1024) return (uint32_t)a * (uint32_t)b / (uint32_t)c;
  return a * b / c;
}

template <int NT, bool WHOLE>
__global__ void __launch_bounds__(THREADS, Shape<NT>::PER_SM) kv4_attention_kernel(const AttnArgs args) {
  constexpr int QT = 8 * NT, STAGES = Shape<NT>::STAGES;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  float* xm = reinterpret_cast<float*>(smem + Shape<NT>::RING);  // [WARPS][QT] maxima, sums; [WARPS][8][CS] outputs
  float* xl = xm + WARPS * QT;
  float* xo = xl + WARPS * QT;
  uint4* sq = reinterpret_cast<uint4*>(smem + Shape<NT>::RING + Shape<NT>::EXCHANGE);  // [NT][4][32]
  uint8_t* srow = reinterpret_cast<uint8_t*>(sq + NT * 128);                           // [2][8 NT][QROW]
  float* ssum = reinterpret_cast<float*>(srow + 2 * QT * QROW);                        // [8 NT][4]
  float* smul = ssum + 32 * NT;                                                        // [8 NT]
  int* spos = reinterpret_cast<int*>(smul + 8 * NT);                                   // [8 NT]
  uint64_t* full = reinterpret_cast<uint64_t*>(spos + 8 * NT);
  int64_t* sums = reinterpret_cast<int64_t*>(full + WARPS * STAGES);  // [WARPS]
  int2* spans = reinterpret_cast<int2*>(sums + WARPS);                // [WARPS]
  Run& run = *reinterpret_cast<Run*>(spans + WARPS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(&run + 1);

  const Seqs& sv = args.seqs;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = warp >> 1, tok0 = HALF * (warp & 1), g = lane >> 2, t = lane & 3;
  const int G = args.HQ / sv.HK;

  if (tid == 0) {
    for (int i = 0; i < WARPS * STAGES; ++i) mbar_init(&full[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  if (tid == 0) pdl_launch();

  // This CTA's run of all items' pages begins at `at`; `sharing` CTAs have one.
  int64_t at = 0, total = 1;
  int sharing = 1;
  if constexpr (WHOLE) {
    if (tid == 0) {
      run.b = blockIdx.x / sv.HK;
      run.item = blockIdx.y;  // the column tile
    }
  } else {
    const int per = (sv.B + THREADS - 1) / THREADS, b_lo = min(tid * per, sv.B), b_hi = min(b_lo + per, sv.B);
    int64_t mine = 0;
    int longest = 0, count = 0;
    for (int i = b_lo; i < b_hi; ++i) {
      const Seq q = seq_at(args, i, QT);
      mine += q.weight(sv.HK);
      count += q.tiles * sv.HK;
      if (q.tiles > 0) longest = max(longest, ITEM_PAGES + q.pages());
    }
    int64_t scan = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, scan, d);
      if (lane >= d) scan += v;
    }
    const int2 span = make_int2(__reduce_max_sync(0xffffffffu, longest), __reduce_add_sync(0xffffffffu, count));
    if (lane == 31) {
      sums[warp] = scan;
      spans[warp] = span;
    }
    __syncthreads();
    int64_t pre = scan - mine;
    int items = 0;
    total = 0;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) pre += sums[w];
      total += sums[w];
      longest = max(longest, spans[w].x);
      items += spans[w].y;
    }
    sharing = (int)max((int64_t)1, min((int64_t)gridDim.x, total / MIN_PAGES));
    if ((int)blockIdx.x >= sharing) return;
    at = mul_div(blockIdx.x, total, sharing);
    int64_t end = mul_div(blockIdx.x + 1, total, sharing);
    // one verdict of all CTAs: end - at is not the same in each
    if (items <= sharing && longest <= APART + mul_div(1, total, sharing)) {  // an item each, none cut
      if ((int)blockIdx.x >= items) return;
      int before = count;
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += v;
      }
      before -= count;
      for (int w = 0; w < warp; ++w) before += spans[w].y;
      int k = (int)blockIdx.x - before;
      if (k >= 0 && k < count) {
        for (int i = b_lo;; ++i) {
          const Seq seq = seq_at(args, i, QT);
          const int n = seq.tiles * sv.HK;
          if (k < n) {
            run.left = ITEM_PAGES + seq.pages();
            run.b = i;
            run.item = k;
            run.from = -ITEM_PAGES;
            break;
          }
          k -= n;
        }
      }
      end = at;  // found
    } else if (at >= end) {
      return;  // no rows at all
    }
    if (at < end && at >= pre && at < pre + mine) {
      int i = b_lo;
      int64_t p = pre;
      for (;; ++i) {
        const Seq seq = seq_at(args, i, QT);
        const int64_t w = seq.weight(sv.HK);
        if (at < p + w) {
          const int span = ITEM_PAGES + seq.pages();
          run.left = end - at;
          run.b = i;
          run.item = (int)(at - p < 0x7fffffff ? (uint32_t)(at - p) / (uint32_t)span : (at - p) / span);
          run.from = (int)(at - p - (int64_t)run.item * span) - ITEM_PAGES;
          break;
        }
        p += w;
      }
    }
  }
  // Finds the CTA's next share; run.more is 0 when there is none.  One thread, which the others wait
  // for: a sequence is looked at once, not once an item.
  auto advance = [&](Share& next) {
    int more = 0, item = run.item, from = run.from, to = 0;
    if constexpr (WHOLE) {
      if (!run.known) {
        run.known = 1;
        run.seq = seq_at(args, run.b, QT);
        run.items = run.seq.tiles;
      }
      more = item < run.items;
      from = 0;
      to = run.seq.pages();
      run.item = item + gridDim.y;
    } else {
      int64_t left = run.left;
      while (left > 0 && !more) {
        if (!run.known || item >= run.items) {
          if (run.known) {
            run.b = run.items > 0 ? run.b + 1 : next_with_rows(sv, run.b);
            if (run.b >= sv.B) left = 0;  // (row_start does not ascend)
            if (left == 0) break;
            item = 0;
            from = -ITEM_PAGES;
          }
          run.known = 1;
          run.seq = seq_at(args, run.b, QT);
          run.items = run.seq.tiles * sv.HK;
          continue;
        }
        to = (int)min((int64_t)run.seq.pages(), from + left);
        left -= to - from;
        more = to > max(from, 0);  // else the run ended in what the item's start stands for
        if (!more) break;
      }
      run.left = left;
      run.item = item + 1;  // or the run is at its end, and left 0
      run.from = -ITEM_PAGES;
    }
    run.more = more;
    if (!more) return;
    const Seq& q = run.seq;
    next.b = run.b;
    next.kvh = WHOLE ? (int)(blockIdx.x % sv.HK) : item % sv.HK;
    next.c0 = (WHOLE ? item : item / sv.HK) * QT;
    next.clast = min(next.c0 + QT, q.S * G) - 1;
    next.i0 = max(from, 0);
    next.i1 = min(to, q.ps.n);
    next.entire = from <= 0 && to == q.pages();
    next.r0 = q.r0;
    next.pos0 = q.ctx - q.S;
    next.ps = q.ps;
    next.pos_lo = next.pos0 + next.c0 / G;
    const int whole_key = args.window > 0 ? max(0, next.pos0 + next.clast / G - args.window + 1) : 0;
    next.whole_lo = q.ps.n_sink + max(0, (whole_key + PAGE - 1) / PAGE - q.ps.first_page);
    next.whole_hi = q.ps.n_sink + min(max(next.pos_lo + 1, 0), q.ps.kend) / PAGE - q.ps.first_page;
    if (q.ctx > sv.max_pages * PAGE) atomicOr(&ffb_device_error_word, (uint32_t)ffb::ERR_KV4_PAGE);
  };

  // This warp's ring: `use` is the stage of its next half page, `fill` the next to load (the same when
  // the ring is full and `use` is done with).  Bit s of `bad`: the page of stage s is outside the cache.
  int use = 0, fill = 0;
  uint32_t use_ph = 0, bad = 0;
  const uint32_t wfull = smem_u32(full + warp * STAGES), wring = smem_u32(smem + warp * STAGES * HALF_BYTES);
  const uint32_t page_bytes = (uint32_t)sv.HK * RECORD;
  // pages i0 + group + GROUPS k of a share are this warp's
  auto pages_in = [&](const Share& s) { return max(0, (s.i1 - s.i0 - group + GROUPS - 1) / GROUPS); };
  auto page_index = [&](const PageSet& ps, int i) { return i < ps.n_sink ? i : ps.first_page + i - ps.n_sink; };
  // lane i: the id of page k + i of the share
  auto ids_from = [&](const Share& s, int k, int cnt) {
    return k + lane < cnt ? __ldg(sv.table + s.b * sv.table_stride + page_index(s.ps, s.i0 + group + GROUPS * (k + lane))) : -1;
  };
  auto load = [&](int page, const uint8_t* head) {  // the whole warp; head: page 0's record of the K/V head
    const uint32_t bar = wfull + 8 * fill, dst = wring + HALF_BYTES * fill;
    if ((uint32_t)page < (uint32_t)sv.num_pages) {
      if (lane == 0) {
        const uint8_t* codes = head + (uint64_t)(uint32_t)page * page_bytes + 64 * tok0;
        const uint8_t* scales = codes - 56 * tok0;
        expect_bytes(bar, HALF_BYTES);
        bulk(dst, codes, HALF_CODES, bar);
        bulk(dst + HALF_KS, scales + K_SCALES, HALF_SCALES, bar);
        bulk(dst + HALF_V, codes + V_CODES, HALF_CODES, bar);
        bulk(dst + HALF_VS, scales + V_SCALES, HALF_SCALES, bar);
      }
    } else {
      bad |= 1u << fill;
      if (lane == 0) {
        atomicOr(&ffb_device_error_word, (uint32_t)ffb::ERR_KV4_PAGE);
        arrive(bar);
      }
    }
    fill = fill + 1 == STAGES ? 0 : fill + 1;
  };
  // where this lane reads in a half page: K codes of token token_of(g), scales, V codes of the
  // tokens of MMA columns 2 t and 2 t + 1
  const int tok_g = token_of(g), k_off = 64 * tok_g + 16 * t, s_off = 8 * tok_g;
  const int v_off = HALF_V + 64 * token_of(2 * t) + 8 * (g ^ (4 * (t >> 1)));
  const int v_next = 64 * (token_of(2 * t + 1) - token_of(2 * t));

  // Brings a share's query rows (column c's is row r0 + c / G of head kvh G + c % G) into shared memory.
  auto fetch_queries = [&](const Share& s, int buffer) {
    if (tid < 16 * QT) {
      const int c = s.c0 + (tid >> 4);
      const bool valid = c <= s.clast;
      const uint16_t* q = args.q + (valid ? ((int64_t)(s.kvh * G + c % G) * sv.T + s.r0 + c / G) * D : 0) + 8 * (tid & 15);
      copy16(srow + (buffer * QT + (tid >> 4)) * QROW + 16 * (tid & 15), q, valid);
    }
  };

  __syncthreads();
  // a replay of a call that gave up may find tags of that run: it gives up too
  if (!WHOLE && tid == 64) run.failed = __ldcg(args.flags + 2 * gridDim.x) == failed_tag(args.tag);
  if (tid == 0) {
    run.cut.b = -1;
    run.known = 0;
    advance(run.share[0]);
  }
  __syncthreads();
  bool more = run.more;
  // of the current share: 32 page ids from page ids_at on, pages in the ring or done
  int ids = -1, ids_at = 0, issued = 0, turn = 0;
  int64_t run_item = at;  // where page 0 of the run's first item lies
  if (more) {
    const Share& first = run.share[0];
    run_item -= first.i0;
    const int cnt = pages_in(first);
    ids = ids_from(first, 0, cnt);
    fetch_queries(first, 0);
    const uint8_t* head = sv.pages + (int64_t)first.kvh * RECORD;
    for (; issued < min(cnt, STAGES); ++issued) load(__shfl_sync(0xffffffffu, ids, issued), head);
  }
  while (more) {
    const Share& cur = run.share[turn];
    copies_done();  // this share's queries
    __syncthreads();
    // the last warp has no query fragments to make (8 columns)
    if (tid == THREADS - 32) advance(run.share[turn ^ 1]);
    if (tid < QT) spos[tid] = cur.c0 + tid <= cur.clast ? cur.pos0 + (cur.c0 + tid) / G : -1;  // the columns' positions
    // query fragments, a warp each: lane (g, t) of (column tile n, scale group j) holds channels
    // 32 j + 8 t .. + 7 of column 8 n + g as the pairs (e, e + 4) that a K word's nibbles come in,
    // scaled into fp16.  Every warp finds the columns' largest values itself.
    if (warp < 4 * NT) {
      const int n = warp >> 2, j = warp & 3;
      const uint8_t* row = srow + (turn * QT + 8 * n + g) * QROW + 16 * t;
      const uint4 x = *reinterpret_cast<const uint4*>(row + 64 * j);
      uint32_t top = 0;  // largest |q| of the column, as bits (a NaN is above infinity)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 y = *reinterpret_cast<const uint4*>(row + 64 * i);
        top = max(max(top, max((y.x << 16) & 0x7fffffffu, y.x & 0x7fff0000u)), max((y.y << 16) & 0x7fffffffu, y.y & 0x7fff0000u));
        top = max(max(top, max((y.z << 16) & 0x7fffffffu, y.z & 0x7fff0000u)), max((y.w << 16) & 0x7fffffffu, y.w & 0x7fff0000u));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^14 <= largest |q| factor < 2^15; a column of infinities or NaN stays one.  A negative
      // scale turns the queries' sign instead
      const int e2 = (int)(top >> 23) - 127, ex = e2 == 128 ? 0 : max(e2, -100);
      const float size = __uint_as_float((uint32_t)(127 + 14 - ex) << 23), factor = args.scale_log2 < 0.f ? -size : size;
      const float q0 = lo_of(x.x) * factor, q1 = hi_of(x.x) * factor, q2 = lo_of(x.y) * factor, q3 = hi_of(x.y) * factor;
      const float q4 = lo_of(x.z) * factor, q5 = hi_of(x.z) * factor, q6 = lo_of(x.w) * factor, q7 = hi_of(x.w) * factor;
      sq[warp * 32 + lane] = make_uint4(pack_f16(q0, q4), pack_f16(q1 * 0.0625f, q5 * 0.0625f), pack_f16(q2, q6),
                                        pack_f16(q3 * 0.0625f, q7 * 0.0625f));
      float sum = ((q0 + q1) + (q2 + q3)) + ((q4 + q5) + (q6 + q7));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == 0) {
        ssum[(8 * n + g) * 4 + j] = sum * -0x1p-21f;  // -8 x 2^-24
        // scores come out 2^-24 factor times too large; beyond 2^110 the (one-hot) softmax only
        // needs their order, as with a factor past 2^116.  Never 0: a masked -inf stays one
        if (j == 0)
          smul[8 * n + g] = fminf(
              fmaxf(fabsf(args.scale_log2) * __uint_as_float((uint32_t)(127 + 10 + min(ex, 110)) << 23), 1e-37f), 0x1p116f);
      }
    }
    __syncthreads();

    // the ids of the next share's first pages, for the stages that this one's last pages leave, and its queries
    more = run.more;
    int next_cnt = 0, next_ids = -1, ahead = 0;
    const uint8_t* next_head = sv.pages;
    if (more) {
      const Share& next = run.share[turn ^ 1];
      next_head += (int64_t)next.kvh * RECORD;
      next_cnt = pages_in(next);
      next_ids = ids_from(next, 0, next_cnt);
      fetch_queries(next, turn ^ 1);
    }
    const PageSet ps = cur.ps;
    const int i0 = cur.i0, whole_lo = cur.whole_lo, whole_hi = cur.whole_hi, cnt = pages_in(cur);
    const uint8_t* head = sv.pages + (int64_t)cur.kvh * RECORD;
    uint2 qo[NT];  // K index 4 part + j of the offsets' MMA: this lane has 2 t, 2 t + 1 and 8 more (part 3: zeros)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float2 u = *reinterpret_cast<const float2*>(ssum + (8 * n + g) * 4 + 2 * (t & 1));
      qo[n] = make_uint2(pack_bf16(bf16_part(u.x, t >> 1), bf16_part(u.y, t >> 1)),
                         t < 2 ? pack_bf16(bf16_part(u.x, 2), bf16_part(u.y, 2)) : 0u);
    }

    float o[8][NT][4];  // O^T, 2^(64 - 133) times too large, 2^4 more in elements 2 and 3
    // of this lane's columns: 64 - maximum, the raw score that moves it, factor, sum 2^64 times too large
    float neg[2 * NT], high[2 * NT], mul[2 * NT], l[2 * NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i][n][e] = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      high[i] = -INFINITY;
      neg[i] = UNSEEN;
      l[i] = 0.f;
      mul[i] = smul[8 * (i >> 1) + 2 * t + (i & 1)];
    }

    // A half page as two fragments of sixteen tokens.  Rows g and g + 8 of fragment f are tokens
    // 16 f + token_of(g) and 8 more.  masked: some column may not see some of them (a branch, not a
    // second copy of the code: what runs once an item is paid in instruction fetches); key0: the
    // first token's position, then.
    auto tokens = [&](const uint8_t* rec, int key0, bool masked) {
      constexpr int F = HALF / 16;
      const uint8_t* kc = rec + k_off;
      const uint8_t* sc = rec + s_off;
      const uint8_t* vc = rec + v_off;
      float s[F][NT][4];
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const uint4 ka = *reinterpret_cast<const uint4*>(kc + 1024 * f);
        const uint4 kb = *reinterpret_cast<const uint4*>(kc + 1024 * f + 8 * 64);
        const uint2 sa = *reinterpret_cast<const uint2*>(sc + HALF_KS + 128 * f);
        const uint2 sb = *reinterpret_cast<const uint2*>(sc + HALF_KS + 128 * f + 8 * 8);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
        const float fa[4] = {lo_of(sa.x), hi_of(sa.x), lo_of(sa.y), hi_of(sa.y)};
        const float fb[4] = {lo_of(sb.x), hi_of(sb.x), lo_of(sb.y), hi_of(sb.y)};
        const uint32_t oa = (t & 1) ? sa.y : sa.x, ob = (t & 1) ? sb.y : sb.x;
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816_0(s[f][n], oa, ob, oa, ob, qo[n].x, qo[n].y);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t va = wa[j] >> 8, vb = wb[j] >> 8;
          const uint32_t a0 = wa[j] & 0x000F000Fu, a1 = wb[j] & 0x000F000Fu, a2 = wa[j] & 0x00F000F0u, a3 = wb[j] & 0x00F000F0u;
          const uint32_t a4 = va & 0x000F000Fu, a5 = vb & 0x000F000Fu, a6 = va & 0x00F000F0u, a7 = vb & 0x00F000F0u;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 q = sq[(n * 4 + j) * 32 + lane];  // (kept in registers they would spill the sums)
            float c[4];
            mma16816_h0(c, a0, a1, a2, a3, q.x, q.y);
            mma16816_h(c, a4, a5, a6, a7, q.z, q.w);
            s[f][n][0] = fmaf(c[0], fa[j], s[f][n][0]);
            s[f][n][1] = fmaf(c[1], fa[j], s[f][n][1]);
            s[f][n][2] = fmaf(c[2], fb[j], s[f][n][2]);
            s[f][n][3] = fmaf(c[3], fb[j], s[f][n][3]);
          }
        }
      }
      if (masked) {
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = key0 + 16 * f + tok_g + (e < 2 ? 0 : 8), p = spos[8 * n + 2 * t + (e & 1)];
              if (key > p || key >= ps.kend || (args.window > 0 && p - key >= args.window && key >= args.sinks))
                s[f][n][e] = -INFINITY;
            }
      }
      bool grow = false;
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) grow |= s[f][n][e] > high[2 * n + (e & 1)];
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
          float x = -INFINITY;
#pragma unroll
          for (int f = 0; f < F; ++f) x = fmaxf(x, fmaxf(s[f][i >> 1][i & 1], s[f][i >> 1][2 + (i & 1)]));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const bool up = x > high[i];
          const float base = smul[8 * (i >> 1) + 2 * t + (i & 1)];
          float to = 64.f - x * mul[i], to_mul = mul[i], a = ex2(to - neg[i]);
          // vast scores, or no longer: an old maximum has no weight beside the new one.  What comes out depends on x
          // alone, so that warps with the same maximum agree
          if (fabsf(x * mul[i]) >= 0x1p30f || to_mul != base) {
            const float small = vast_scale(x * base);
            to_mul = base * small;
            to = (small == 1.f ? 64.f : 32.f) - x * to_mul;
            a = to_mul == mul[i] ? ex2(to - neg[i]) : 0.f;
          }
          if (!up) continue;
          neg[i] = to;
          mul[i] = to_mul;
          high[i] = x + __fdividef(LAZY, to_mul);
          l[i] *= a;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            o[d][i >> 1][i & 1] *= a;
            o[d][i >> 1][2 + (i & 1)] *= a;
          }
        }
      }
#pragma unroll
      for (int f = 0; f < F; ++f) {
        uint32_t pb[NT][8];  // P^T fragments, V's scale of group j folded in
        const uint2 sa = *reinterpret_cast<const uint2*>(sc + HALF_VS + 128 * f);
        const uint2 sb = *reinterpret_cast<const uint2*>(sc + HALF_VS + 128 * f + 8 * 8);
        const float fa[4] = {lo_of(sa.x), hi_of(sa.x), lo_of(sa.y), hi_of(sa.y)};
        const float fb[4] = {lo_of(sb.x), hi_of(sb.x), lo_of(sb.y), hi_of(sb.y)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 2 * n + (e & 1);
            // neg stays finite until the first score: -inf gives 0 in every case
            p[e] = ex2(fmaf(s[f][n][e], mul[i], neg[i]));
            l[i] += p[e];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 y02 = mul_pair(p[0], p[2], fa[j], fb[j]), y13 = mul_pair(p[1], p[3], fa[j], fb[j]);
            pb[n][2 * j] = pack_bf16(y02.x, y13.x);
            pb[n][2 * j + 1] = pack_bf16(y02.y, y13.y);
          }
          if (masked) {  // nothing of a masked token counts, whatever its scale holds; one that is seen counts at p = 0 too
            const float(&x)[4] = s[f][n];
            const uint32_t ka = (x[0] == -INFINITY ? 0u : 0xffffu) | (x[1] == -INFINITY ? 0u : 0xffff0000u);
            const uint32_t kb = (x[2] == -INFINITY ? 0u : 0xffffu) | (x[3] == -INFINITY ? 0u : 0xffff0000u);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              pb[n][2 * j] &= ka;
              pb[n][2 * j + 1] &= kb;
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) pb[n][j] = transpose8x8(pb[n][j]);
        }
        // V^T fragments: columns 2t, 2t+1, 2t+8, 2t+9 of the MMA are these four tokens
        const uint8_t* v = vc + 1024 * f;
        const uint2 v0 = *reinterpret_cast<const uint2*>(v), v1 = *reinterpret_cast<const uint2*>(v + v_next);
        const uint2 v2 = *reinterpret_cast<const uint2*>(v + 512), v3 = *reinterpret_cast<const uint2*>(v + v_next + 512);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t x0 = half ? v0.y : v0.x, x1 = half ? v1.y : v1.x, x2 = half ? v2.y : v2.x, x3 = half ? v3.y : v3.x;
#pragma unroll
          for (int quart = 0; quart < 2; ++quart) {
            const uint32_t sel = quart ? 0x7632 : 0x5410;
            uint32_t lo = __byte_perm(x0, x1, sel), hi = __byte_perm(x2, x3, sel);  // tokens (2t, 2t+1), (2t+8, 2t+9)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int mt = 4 * half + 2 * quart + u;  // channels 16 mt + g and (sixteen times too large) 16 mt + 8 + g
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint32_t p0 = pb[n][2 * (mt >> 1)], p1 = pb[n][2 * (mt >> 1) + 1];
                mma16816(o[mt][n], lo & 0x000F000Fu, lo & 0x00F000F0u, hi & 0x000F000Fu, hi & 0x00F000F0u, p0, p1);
                mma16816(o[mt][n], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, p0, p1);
              }
              lo >>= 8;
              hi >>= 8;
            }
          }
        }
      }
    };

    bool ok = true;
    for (int k = 0; k < cnt; ++k) {
      // one verdict for the warp: its lanes stay together whatever each of them saw
      if (!__all_sync(0xffffffffu, arrived(wfull + 8 * use, use_ph)) &&
          !__all_sync(0xffffffffu, mbar_wait_bounded(full + warp * STAGES + use, use_ph, abort_flag))) {
        ok = false;
        break;
      }
      if (!((bad >> use) & 1u)) {
        const int i = i0 + group + GROUPS * k;
        const bool masked = i < whole_lo || i >= whole_hi;
        int key0 = 0;
        if (masked) key0 = page_index(ps, i) * PAGE + tok0;
        if (!masked || key0 < ps.kend) tokens(smem + (warp * STAGES + use) * HALF_BYTES, key0, masked);
      } else {
        bad &= ~(1u << use);
      }
      __syncwarp();  // every lane has read the stage
      if (issued < cnt) {
        if (issued - ids_at == 32) {
          ids_at = issued;
          ids = ids_from(cur, ids_at, cnt);
        }
        load(__shfl_sync(0xffffffffu, ids, issued - ids_at), head);
        ++issued;
      } else if (ahead < next_cnt) {
        load(__shfl_sync(0xffffffffu, next_ids, ahead), next_head);
        ++ahead;
      }
      if (++use == STAGES) {
        use = 0;
        use_ph ^= 1u;
      }
    }
    if (!ok) *abort_flag = 1;
    // a share with fewer pages than stages leaves some of the ring's to fill
    for (; ahead < min(next_cnt, STAGES) && !__any_sync(0xffffffffu, *abort_flag); ++ahead)
      load(__shfl_sync(0xffffffffu, next_ids, ahead), next_head);
    issued = ahead;
    ids = next_ids;
    ids_at = 0;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
      if (g == 0) {
        const int c = 8 * (i >> 1) + 2 * t + (i & 1);
        xm[warp * QT + c] = neg[i] == UNSEEN ? -INFINITY : mul[i] == smul[c] ? 64.f - neg[i] : (64.f - neg[i]) * (smul[c] / mul[i]);
        xl[warp * QT + c] = l[i] * 0x1p-64f;
      }
    }
    // the warps' sums, eight columns at a time
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (n > 0) __syncthreads();
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        float* dst = xo + (warp * 8 + 2 * t) * CS + 16 * mt + g;
        dst[0] = o[mt][n][0] * 0x1p69f;
        dst[CS] = o[mt][n][1] * 0x1p69f;
        dst[8] = o[mt][n][2] * 0x1p65f;
        dst[CS + 8] = o[mt][n][3] * 0x1p65f;
      }
      __syncthreads();
      // 8 columns x 128 channels over 256 threads: four neighbouring channels a thread, a warp a column
      const int c = warp, d = 4 * lane;
      const int col = cur.c0 + 8 * n + c;
      if (col <= cur.clast) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, xm[w * QT + 8 * n + c]);
        float sum = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int w = 0; w < WARPS; ++w) {
          const float mw = xm[w * QT + 8 * n + c], lw = xl[w * QT + 8 * n + c];
          if (mw == -INFINITY && lw == 0.f) continue;  // this warp saw nothing of the row
          const float f = ex2(mw - top);
          const float4 v = *reinterpret_cast<const float4*>(xo + (w * 8 + c) * CS + d);
          sum = fmaf(lw, f, sum);
          y.x = fmaf(v.x, f, y.x);
          y.y = fmaf(v.y, f, y.y);
          y.z = fmaf(v.z, f, y.z);
          y.w = fmaf(v.w, f, y.w);
        }
        const int row = cur.r0 + col / G, h = cur.kvh * G + col % G;
        if (cur.entire) {
          const float r = sum == 0.f ? 0.f : 1.f / sum;  // nothing visible: zeros
          *reinterpret_cast<uint2*>(args.out + ((int64_t)row * args.HQ + h) * D + d) =
              make_uint2(pack_bf16(y.x * r, y.y * r), pack_bf16(y.z * r, y.w * r));
        } else {  // slot 0: an item that began in a CTA before this one; slot 1: one that begins here
          const int64_t pt = ((int64_t)blockIdx.x * 2 + (i0 == 0)) * QT + 8 * n + c;
          *reinterpret_cast<float4*>(args.part_o + pt * D + d) = y;
          if (lane == 0) *reinterpret_cast<float2*>(args.part_ml + pt * 2) = make_float2(top, sum);
          __threadfence();
        }
      }
    }
    // before the next share overwrites the exchange; one verdict for the CTA
    if (__syncthreads_or(*abort_flag)) break;
    if (!cur.entire && tid == 0) {
      if (i0 > 0 && cur.i1 == ps.n) run.cut = cur;
      else st_release_gpu_u64(args.flags + 2 * blockIdx.x + (i0 == 0), args.tag);
    }
    turn ^= 1;
  }
  copies_done();
  // A wait that gave up: every warp's copies in flight land before the CTA leaves, those of the warps that
  // had loaded the next share's first pages by then too.  (The flag is the same for all since the last barrier.)
  if (lane == 0 && *abort_flag) {
    volatile int never = 0;
    for (int i = 0; i < STAGES; ++i) {
      mbar_wait_bounded(full + warp * STAGES + i, 0, &never, 20000000ull);
      mbar_wait_bounded(full + warp * STAGES + i, 1, &never, 20000000ull);
    }
  }
  if (!WHOLE && !__syncthreads_or(*abort_flag) && run.cut.b >= 0) {
    const Share& cut = run.cut;
    // The parts of the item that this CTA's first share ended: those of the CTAs from `c_lo` on.  They
    // come before this one, so they run or have run; each puts the call's tag into its flag once its
    // part is written, and this CTA takes the tags off again for the next replay of the call.
    const int c_lo = (int)(((run_item + 1) * sharing - 1) / total), me = blockIdx.x;
    bool ready = true;
    for (int c = c_lo + lane; c < me; c += 32) {
      const uint64_t t0 = global_timer_ns();
      while (ld_acquire_gpu_u64(args.flags + 2 * c + (c == c_lo)) != args.tag) {
        if (global_timer_ns() - t0 > 2000000000ull) {
          ready = false;
          break;
        }
      }
    }
    ready = __all_sync(0xffffffffu, ready) && !run.failed;
    if (!ready) *abort_flag = 1;
    // `side` warps a column, each with every side-th part: a lane finds a part's weight, then the rows
    // are read with nothing in between
    const int cols = cut.clast + 1 - cut.c0, side = cols <= 2 ? 4 : cols <= 4 ? 2 : 1, sub = warp % side;
    Sum* shares = reinterpret_cast<Sum*>(smem);  // [WARPS][32], over the ring
    for (int c1 = 0; c1 < cols; c1 += WARPS / side) {
      const int col = c1 + warp / side;
      Sum s = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
      if (col < cols && ready) {
        for (int first = c_lo + sub; first <= me; first += 32 * side) {
          const int mine = first + lane * side;
          const int64_t pt = ((int64_t)mine * 2 + (mine == c_lo)) * QT + col;
          float2 ml = make_float2(-INFINITY, 0.f);
          if (mine <= me) ml = __ldcg(reinterpret_cast<const float2*>(args.part_ml + pt * 2));
          const float top = fmaxf(s.top, warp_max(ml.x));
          const bool any = !(ml.x == -INFINITY && ml.y == 0.f);  // of the row was seen there
          const uint32_t seen = __ballot_sync(0xffffffffu, any);
          const float f = any ? ex2(ml.x - top) : 0.f, fs = s.top == top ? 1.f : ex2(s.top - top);
          s.l = fmaf(s.l, fs, warp_sum(ml.y * f));
          s.o = make_float4(s.o.x * fs, s.o.y * fs, s.o.z * fs, s.o.w * fs);
          s.top = top;
          const int count = min(32, (me - first) / side + 1);
#pragma unroll 8
          for (int i = 0; i < count; ++i) {
            const int part = first + i * side;
            const float4 v = __ldcg(reinterpret_cast<const float4*>(
                args.part_o + (((int64_t)part * 2 + (part == c_lo)) * QT + col) * D + 4 * lane));
            const float w = __shfl_sync(0xffffffffu, f, i);
            if (seen >> i & 1u) {  // a part that saw nothing may hold anything; NaN of no weight is NaN
              s.o.x = fmaf(v.x, w, s.o.x);
              s.o.y = fmaf(v.y, w, s.o.y);
              s.o.z = fmaf(v.z, w, s.o.z);
              s.o.w = fmaf(v.w, w, s.o.w);
            }
          }
        }
      }
      if (side > 1) {
        __syncthreads();
        shares[warp * 32 + lane] = s;
        __syncthreads();
        if (sub == 0)
          for (int w = 1; w < side; ++w) {
            const Sum& x = shares[(warp + w) * 32 + lane];
            add_part(s, x.top, x.l, x.o);
          }
      }
      const int c = cut.c0 + col;
      if (sub == 0 && col < cols && ready)
        store_row(args.out + ((int64_t)(cut.r0 + c / G) * args.HQ + cut.kvh * G + c % G) * D, s, lane);
    }
    __syncthreads();
    for (int c = c_lo + tid; c < me; c += THREADS) args.flags[2 * c + (c == c_lo)] = 0;
  }
  if (tid == 0 && *abort_flag) {
    atomicOr(&ffb_device_error_word, (uint32_t)ffb::ERR_ATTN_TIMEOUT);
    if (!WHOLE) args.flags[2 * gridDim.x] = failed_tag(args.tag);
  }
}

// Joins the shares of attention_kv4_tc.cu: 16 CTAs an item that was cut, 32 rows and 64 channels each.
// Channel 64 half + 8 i + g of a row sits in column 16 g + 8 half + 2 (i % 4) + i / 4 of its sums, and
// columns 4 k .. 4 k + 3 of all 256 rows lie next to each other: warp g takes k = 4 g + 2 half and the
// next, a lane a row, and the rows leave through shared memory.
__global__ void __launch_bounds__(256) kv4_join_tc_kernel(const AttnArgs args) {
  __shared__ uint16_t sh[32][66];
  pdl_wait();
  pdl_launch();
  const int cut = (int)(blockIdx.x >> 4), first = (int)(blockIdx.x >> 1 & 7) * 32, half = (int)(blockIdx.x & 1);
  const int g = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TcItem item = tc_item(args, cut);
  const int G = args.HQ / args.seqs.HK, c0 = item.tile * 256 + first, n = min(item.rows * G - c0, 32);  // rows here
  if (n <= 0) return;
  const int row = first + min(lane, n - 1);
  Sum s[2];
  for (int e = 0; e < 2; ++e) s[e] = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
  for (int p = 0; p < args.splits; ++p) {
    const int64_t part = (int64_t)cut * args.splits + p;
    const float2 ml = *reinterpret_cast<const float2*>(args.part_ml + (part * 256 + row) * 2);
    const float4* from = reinterpret_cast<const float4*>(args.part_o) + (part * (D / 4) + 4 * g + 2 * half) * 256 + row;
    const float4 v0 = from[0], v1 = from[256];
    add_part(s[0], ml.x, ml.y, v0);
    add_part(s[1], ml.x, ml.y, v1);
  }
  const float r = s[0].l == 0.f ? 0.f : 1.f / s[0].l;
  for (int e = 0; e < 2; ++e) {  // columns 4 e .. of eight: i = 2 e, 2 e + 4, 2 e + 1, 2 e + 5
    const uint32_t lo = pack_bf16(s[e].o.x * r, s[e].o.y * r), hi = pack_bf16(s[e].o.z * r, s[e].o.w * r);
    sh[lane][8 * (2 * e) + g] = (uint16_t)lo;
    sh[lane][8 * (2 * e + 4) + g] = (uint16_t)(lo >> 16);
    sh[lane][8 * (2 * e + 1) + g] = (uint16_t)hi;
    sh[lane][8 * (2 * e + 5) + g] = (uint16_t)(hi >> 16);
  }
  __syncthreads();
  for (int k = g; k < n; k += 8) {
    const int c = c0 + k;
    uint32_t* to = reinterpret_cast<uint32_t*>(args.out + ((int64_t)(item.r0 + c / G) * args.HQ + item.kvh * G + c % G) * D);
    to[32 * half + lane] = *reinterpret_cast<const uint32_t*>(&sh[k][2 * lane]);
  }
}

// How a call is laid out.  kernel: 1 / 2 = the register path with 8 / 16 query columns a CTA,
// TC = the tensor-memory path with 256.  splits: the shares of the pages of each of TC's first
// `cut` items, behind which come `whole` items of one CTA; the register path has 1 (every item one
// CTA's) or 0 (all pages in equal runs).
constexpr int TC = 3;
struct Plan {
  int kernel, tiles, splits, ctas, cut, whole;
  int64_t bytes;  // workspace
};

// TC: whole items while they fill every SM, the rest (or all) in shares that fill the last wave.
// The costs in us: a block of two pages 2.2, a CTA's start and end 10, the join's launch 2, a cut
// item's share of partial sums written and read 0.07.
constexpr double BLOCK_US = 2.2, CTA_US = 10.0, JOIN_US = 2.0, SHARE_US = 0.07;
void plan_tc(Plan& p, int64_t items, int64_t pages, int sms) {
  const int64_t blocks = (pages + 1) / 2;
  const double item_us = (double)blocks * BLOCK_US + CTA_US;
  double best = 0;
  auto look = [&](int64_t whole, int64_t splits) {
    if (splits < 1 || splits > 64 || (splits > 1 && splits > blocks)) return;
    const int64_t shares = (items - whole) * splits;
    const double cost = (double)(whole / sms) * item_us +
                        (double)((shares + sms - 1) / sms) * ((double)((blocks + splits - 1) / splits) * BLOCK_US + CTA_US) +
                        (splits > 1 ? JOIN_US + SHARE_US * (double)shares : 0.0);
    if (best == 0 || cost < best) {
      best = cost;
      p.splits = (int)splits;
      p.whole = splits > 1 ? (int)whole : (int)items;
      p.cut = (int)items - p.whole;
    }
  };
  const int64_t full = items / sms * sms;
  for (int64_t whole = full; whole >= 0 && whole >= full - sms; whole -= sms) {
    look(whole, 1);
    if (whole == items) continue;
    for (int wave = 1; wave <= 3; ++wave) look(whole, wave * sms / (items - whole));
    for (int64_t n = 1; n <= 6; ++n) look(whole, (blocks + n - 1) / n);  // shares of n blocks
  }
  p.ctas = p.whole + p.cut * p.splits;
  p.bytes = (int64_t)p.cut * p.splits * 256 * (D + 2) * 4;
}

Plan make_plan(int B, int T, int HQ, int HK, int max_rows, int max_pages, int window, int sinks) {
  Plan p;
  const int64_t cols = (int64_t)max_rows * (HQ / HK);
  // 8 columns a CTA, 16, or 256 of tensor memory.  us with each, 16 sequences of 8192 tokens, 32 + 8
  // heads: 4 columns 49 / 71 / 133, 16 columns 84 / 76 / 137, 24 columns 119 / 134 / 140, 32 columns
  // 154 / 135 / 143, 48 columns 222 / 193 / 143.
  p.kernel = cols > 32 ? TC : cols <= 8 || (cols > 16 && cols <= 24) ? 1 : 2;
  const int width = p.kernel == TC ? 256 : 8 * p.kernel;
  const int64_t tiles = (cols + width - 1) / width;
  p.tiles = (int)(tiles < 4096 ? tiles : 4096);
  int64_t pages = max_pages;
  if (window > 0) {
    const int64_t seen = ((int64_t)sinks + 63) / 64 + ((int64_t)window + max_rows + 126) / 64;
    if (seen < pages) pages = seen;
  }
  const int sms = ffb::sm_count();
  if (p.kernel == TC) {
    // the tiles of all sequences: each has max_rows at most, together they have T
    const int64_t all = (int64_t)T * (HQ / HK) / 256 + B;
    plan_tc(p, (int64_t)HK * (all < B * tiles ? all : B * tiles), pages, sms);
  } else {
    // Narrow tables: each item one CTA's, without a look at all lengths.  us so / in runs, 32 + 8 heads: one
    // sequence of 1024 tokens 11.6 / 12.3, of 1536 14.5 / 13.0; 8 of 1536 15.1 / 16.4, of 2048 17.8 / 17.8;
    // 128 of 2048 86 / 93; 32 of 300 to 2048 in one call 23.9 / 24.6.
    p.splits = pages <= (B * HK * tiles >= 64 ? 32 : 16) ? 1 : 0;
    p.cut = p.whole = 0;
    p.ctas = p.splits ? B * HK : sms * (p.kernel == 1 ? Shape<1>::PER_SM : Shape<2>::PER_SM);
    p.bytes = p.splits ? 0 : (int64_t)p.ctas * 2 * (8 + width * (D + 2) * 4) + 128;
  }
  return p;
}

// A number that no memory holds by chance and no other call uses: what marks a call's parts as
// written in a workspace that nothing cleared.
uint64_t call_tag() {
  static std::atomic<uint64_t> calls{(uint64_t)std::chrono::steady_clock::now().time_since_epoch().count() << 20};
  uint64_t x = calls.fetch_add(1) * 0x9E3779B97F4A7C15ull;
  x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
  x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
  return (x ^ (x >> 31)) | 1;
}

template <int NT>
cudaError_t launch_registers(const Plan& p, const AttnArgs& a, cudaStream_t st) {
  void (*kernel)(const AttnArgs) = p.splits ? kv4_attention_kernel<NT, true> : kv4_attention_kernel<NT, false>;
  cudaError_t e = ffb::set_smem_attr(reinterpret_cast<const void*>(kernel), Shape<NT>::SMEM);
  if (e == cudaSuccess)
    e = ffb::launch(kernel, dim3(p.ctas, p.splits ? p.tiles : 1), dim3(THREADS), Shape<NT>::SMEM, st, a);
  return e;
}

}  // namespace

namespace kv4 {
cudaError_t launch_attention_tc(const AttnArgs& a, unsigned ctas, cudaStream_t stream);
}

extern "C" int64_t ffb_attention_kv4_workspace(int B, int T, int HQ, int HK, int max_rows, int max_pages, int window,
                                               int sinks) {
  if (B <= 0 || T <= 0 || HQ <= 0 || HK <= 0 || HQ % HK != 0 || max_rows <= 0 || max_pages <= 0 || window < 0 || sinks < 0)
    return 0;
  if (B > 65535 || T > (1 << 24) || HK > 1024 || HQ > 4096 || (int64_t)T * HQ > (1 << 30) || max_rows > T ||
      max_pages > FFB_KV4_MAX_PAGES || window > (1 << 30) || sinks > (1 << 30))
    return 0;  // what the call refuses: the plan's products are made for less
  return make_plan(B, T, HQ, HK, max_rows, max_pages, window, sinks).bytes;
}

extern "C" int ffb_attention_kv4(const uint16_t* q, const uint8_t* pages, int num_pages, const int* page_table,
                                 int64_t table_stride, int max_pages, const int* row_start, const int* ctx_len,
                                 uint16_t* out, void* ws, int64_t ws_bytes, int B, int T, int max_rows, int HQ, int HK,
                                 float scale, int window, int sinks, void* stream) {
  const char* who = "ffb_attention_kv4";
  int rc = ffb::kv4_check(who, pages, page_table, row_start, ctx_len, num_pages, table_stride, max_pages, B, T, HK);
  if (rc) return rc;
  FFB_REQUIRE(q && out, "%s: NULL pointer", who);
  FFB_REQUIRE(HQ > 0 && HQ % HK == 0 && HQ <= 4096, "%s: bad heads HQ=%d HK=%d", who, HQ, HK);
  FFB_REQUIRE(max_rows > 0 && max_rows <= T, "%s: max_rows %d (1..T=%d)", who, max_rows, T);
  FFB_REQUIRE(isfinite(scale * LOG2E), "%s: scale %g (times log2 e it must be finite)", who, (double)scale);
  FFB_REQUIRE(window >= 0 && sinks >= 0 && window <= (1 << 30) && sinks <= (1 << 30), "%s: window %d, sinks %d", who,
              window, sinks);
  FFB_REQUIRE((int64_t)T * HQ <= (1 << 30), "%s: T=%d x HQ=%d too large", who, T, HQ);
  FFB_REQUIRE(sinks == 0 || window > 0, "%s: sinks without a window", who);
  FFB_REQUIRE(ffb::aligned(q, 16) && ffb::aligned(out, 16), "%s: q and out must be 16-byte aligned", who);
  const Plan p = make_plan(B, T, HQ, HK, max_rows, max_pages, window, sinks);
  FFB_REQUIRE(p.bytes == 0 || (ws && ws_bytes >= p.bytes && ffb::aligned(ws, 16)),
              "%s: workspace of %lld bytes (16-byte aligned) needed, %lld given", who, (long long)p.bytes, (long long)ws_bytes);
  const int64_t bytes = (int64_t)T * HQ * D * 2;
  FFB_REQUIRE(((T == 1 || HQ == 1) && out == q) || !ffb::overlap(q, bytes, out, bytes), "%s: q and out overlap", who);
  AttnArgs a = {q, out, nullptr, 0, nullptr, nullptr,
                {const_cast<uint8_t*>(pages), page_table, row_start, ctx_len, num_pages, max_pages, B, T, HK, table_stride},
                HQ, p.splits, window, sinks, p.whole, p.cut, scale * LOG2E, nullptr};
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (p.kernel == TC) {
    e = cudaGetSymbolAddress(reinterpret_cast<void**>(&a.errors), ffb_device_error_word);
    if (e != cudaSuccess) return ffb::fail(FFB_ECUDA, "%s: %s", who, cudaGetErrorString(e));
    a.part_o = static_cast<float*>(ws);
    a.part_ml = a.part_o + (int64_t)p.cut * p.splits * 256 * D;
    e = kv4::launch_attention_tc(a, (unsigned)p.ctas, st);
    if (e == cudaSuccess && p.cut > 0) e = ffb::launch(kv4_join_tc_kernel, dim3((unsigned)p.cut * 16), dim3(256), 0, st, a);
  } else {
    // flags and the mark of a failed run (128 bytes, so that rows stay on their lines: off them 131001 tokens
    // take 50.5 us instead of 48.3), partial rows, their maxima and sums
    if (!p.splits) {
      a.flags = static_cast<uint64_t*>(ws);
      a.tag = call_tag();
      a.part_o = reinterpret_cast<float*>(a.flags + 2 * p.ctas + 16);
      a.part_ml = a.part_o + (int64_t)p.ctas * 2 * 8 * p.kernel * D;
    }
    e = p.kernel == 1 ? launch_registers<1>(p, a, st) : launch_registers<2>(p, a, st);
  }
  if (e != cudaSuccess) return ffb::fail(FFB_ECUDA, "%s: %s", who, cudaGetErrorString(e));
  return FFB_OK;
}
