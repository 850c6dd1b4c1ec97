// Attention over the 4-bit paged K/V cache for many query rows a sequence (questions of tens
// of rows over a cached prefix, chunks of hundreds), on tcgen05 with the codes dequantised in
// shared memory.  Semantics and arguments: attention_kv4.cu, which plans and launches it.
//
// One CTA takes an item, 256 query columns ((row, head of the group) pairs of one K/V head; two MMA
// tiles of 128, A and B), or a share of its visible pages, two pages (128 keys) a block:
//   warp 0       finds the item; raw producer: one bulk copy of 9216 bytes a page into a ring
//   warp 1       tensor memory, and the MMAs:
//                S = Q K^T (M 128, N 128, 8 steps of 16 channels), O += P V (8 steps of 16 keys,
//                P read from tensor memory, V row-major)
//   warps 4-11   softmax: four warps a tile, one thread a row
//   warps 12-19  dequantisation: codes and scales of a block -> K and V tiles in bf16 (exact:
//                five bits times three), 128-byte swizzled, in a ring of three 32 KB slots
// The dequantisation is paid once per 256 columns, which is what makes the tensor cores worth
// it over the register path of attention_kv4.cu.  Two query tiles let the MMAs of one run
// while the other is in its softmax; the product of a page starts when its probabilities are there.
// Tensor memory: S_A, S_B, O_A, O_B of 128 columns each; P (bf16) overwrites the first 64 columns of
// its S.
//
// The running maximum of a row moves only when a score passes it by more than 8 (base 2), so
// O stays in tensor memory and is rescaled there by the softmax warps on those rare blocks.
// Channels are permuted inside the MMAs, never in memory: eight channels of a K word come out
// of the nibble pairs as 0 4 1 5 2 6 3 7 and Q is laid out the same; the columns of O are
// taken back to channels when they are stored.
// A token whose V scale is not finite would poison rows that may not see it (0 x NaN), so its
// V row is written as zeros and its K row as NaN: exactly the rows that see it become NaN.
//
// Measured, 512 rows of each of four sequences over 8704 tokens, 64 + 8 heads: 590 us, 960 TFLOP/s, in short
// runs; 641 us, 885 TFLOP/s, called over and over (the clocks fall under the power limit).
// The same walk with the MMAs alone takes 422 us, with the dequantisation 454, with the softmax 540: the
// MMAs' operands in shared memory bound it first (a block of both tiles reads 192 KB there), then the
// chain S -> maximum -> exp -> P -> O of a tile, 2400 of a block's 3800 clocks beside 1200 of waiting
// for S.  64 rows over 2112 tokens, 32 + 8 heads: 23 us, of which 5 until the first S and 8 for storing
// the shares and their join.  Tried and slower: blocks of 64 keys with S held twice (653 us: an MMA
// of N 64 costs as much as one of 128), four warps for K and four for V (631), a fourth slot for three
// raw pages (618), a row's scores kept in registers beside four dequantising warps (668), some of
// the exponentials on the multiply-add pipe (an eighth no gain, a quarter 4% slower).
#include "kv4.cuh"
#include "pdl.cuh"

namespace {

using namespace kv4;

constexpr int DEQUANT = 8;              // warps
constexpr int THREADS = 384 + 32 * DEQUANT;
// Registers a thread by role (warps 0-3, 4-11, 12-19), out of the LAUNCH_REGS x THREADS of the launch:
// what a role gives up, setmaxnreg.dec, the softmax takes, setmaxnreg.inc (which waits for them).
constexpr int LAUNCH_REGS = 96, REGS_ISSUE = 88, REGS_SOFTMAX = 112, REGS_DEQUANT = 80;
static_assert(REGS_ISSUE <= LAUNCH_REGS && REGS_DEQUANT <= LAUNCH_REGS && REGS_SOFTMAX >= LAUNCH_REGS, "wrong way");
static_assert(128 * REGS_ISSUE + 256 * REGS_SOFTMAX + 32 * DEQUANT * REGS_DEQUANT <= LAUNCH_REGS * THREADS, "too many");
constexpr int RAW = 6;                 // raw pages in flight
constexpr int SLOTS = 3;               // 128-key K or V tiles
constexpr int HALF = 128 * 128;        // 64 channels (K, Q) or columns (V) of 128 rows: 16 KB
constexpr int TILE = 2 * HALF;
constexpr int SMEM = 2 * TILE + SLOTS * TILE + RAW * RECORD + 512 + 1024;
constexpr float LAZY = 8.f;

// D[tmem] (+)= A[tmem] B[smem]^T, bf16.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One thread of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
// fp32 pairs in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 u, v, w;\n\t"
      "mov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\t"
      "fma.rn.f32x2 u, u, v, w;\n\tmov.b64 {%0, %1}, u;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 u, v;\n\t"
      "mov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %5};\n\t"
      "add.rn.f32x2 u, u, v;\n\tmov.b64 {%0, %1}, u;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r =
      __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// The eight codes of a word times the scale pair s, in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ uint4 dequant8(uint32_t w, uint32_t s) {
  return make_uint4(mul2(minus136(pair136(w, 0)), s), mul2(minus136(pair136(w, 1)), s), mul2(minus136(pair136(w, 2)), s),
                    mul2(minus136(pair136(w, 3)), s));
}
__device__ __forceinline__ bool not_finite2(uint32_t w) {  // either bf16 of the pair
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
// The channel of column (chunk, pos) of O: chunk = 2 g + half holds nibbles of V's chunk g.
__device__ __forceinline__ int nibble_of(int pos) { return (pos >> 1) | ((pos & 1) << 2); }

// What a CTA does next: shared by its roles, so that it takes no registers of theirs.
struct Work {
  const int* table;
  int kvh, r0, c0, clast;  // K/V head (-1: nothing more), first row, first and last column
  int ctx, first_pos;      // tokens held; the position of the sequence's first row
  int pos_lo, pos_hi;      // of the columns
  int i0, i1, parts;       // its pages of ps, and how many shares those are of
  int seen0, seen1;        // its blocks seen0 .. seen1 - 1: every column sees every key (sinks aside)
  PageSet ps;
  __device__ __forceinline__ int blocks() const { return (i1 - i0 + 1) / 2; }
  __device__ __forceinline__ int page_index(int i) const { return i < ps.n_sink ? i : ps.first_page + i - ps.n_sink; }
};

__global__ void __launch_bounds__(THREADS, 1) kv4_attention_tc_kernel(const AttnArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;                    // Q tiles A, B (at the end: the staged output rows)
  uint8_t* slots = sq + 2 * TILE;
  uint8_t* raw = slots + SLOTS * TILE;
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(raw + RAW * RECORD);
  uint64_t* raw_empty = raw_full + RAW;
  uint64_t* slot_full = raw_empty + RAW;
  uint64_t* slot_empty = slot_full + SLOTS;
  uint64_t* q_full = slot_empty + SLOTS;  // [2] per tile, as the rest
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = s_full + 2;  // [2][2]: the first and the second page's probabilities
  uint64_t* o_done = p_full + 4;
  uint64_t* last = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(last + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* raw_bad = abort_flag + 1;  // [RAW]: the page is absent or its id outside the cache
  // [16] the same of the pages of block u, two bits: what the softmax of that block masks.  It follows
  // the producer through the pages' and tiles' barriers by at most eight blocks.
  volatile int* blk_bad = raw_bad + RAW;
  Work* work = reinterpret_cast<Work*>(smem + 2 * TILE + SLOTS * TILE + RAW * RECORD + 384);

  const Seqs& sv = args.seqs;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = args.HQ / sv.HK;

  if (tid == 0) {
    for (int i = 0; i < RAW; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], DEQUANT);
    }
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&slot_full[i], DEQUANT);
      mbar_init(&slot_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(last, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's, so they start at 0
  pdl_wait();
  if (tid == 0) pdl_launch();

  // Every role takes the same items one after the other; its counters run over all of them.
  uint32_t blk0 = 0;               // blocks of the items before this one
  uint32_t blkB0 = 0;              // those of them that tile B took part in
  uint32_t tiles = 0, tilesB = 0;  // items with blocks
  bool ok = true;
  // The first `whole` CTAs do an item each, those behind them one of `splits` shares of the pages of
  // an item.  If the sequences have more items than the call was laid out for, those that began an
  // item go on with them, uncut.
  auto find_work = [&](int step) {
    const int share = (int)blockIdx.x - args.whole, split = share < 0 ? 0 : share % args.splits;
    const int n = (share < 0 ? args.cut + (int)blockIdx.x : share / args.splits) + step * (args.cut + args.whole);
    const int parts = share < 0 || step > 0 ? 1 : args.splits;
    const TcItem item = tc_item(args, n);
    if (lane == 0) {
      Work w;
      w.kvh = item.r0 < 0 || split >= parts ? -1 : item.kvh;
      w.table = sv.table + item.b * sv.table_stride;
      w.r0 = item.r0;
      w.c0 = item.tile * 256;
      w.clast = min(w.c0 + 256, item.rows * G) - 1;
      w.ctx = item.ctx;
      w.first_pos = item.ctx - item.rows;
      w.pos_lo = w.first_pos + w.c0 / G;
      w.pos_hi = w.first_pos + w.clast / G;
      w.ps = pages_of(w.pos_lo, w.pos_hi, sv.max_pages, args.window, args.sinks);
      const int pairs = (w.ps.n + 1) / 2;
      w.i0 = 2 * (int)((int64_t)split * pairs / parts);
      w.i1 = min(2 * (int)((int64_t)(split + 1) * pairs / parts), w.ps.n);
      w.parts = parts;
      // pages from .. to - 1 are seen whole by all columns
      const int from = args.window > 0 ? max(w.pos_hi - args.window + PAGE, 0) / PAGE : 0;
      const int to = min(w.pos_lo + 1, w.ps.kend) / PAGE, shift = w.ps.n_sink - w.ps.first_page - w.i0;
      w.seen0 = (max(from + shift, w.ps.n_sink - w.i0) + 1) >> 1;
      w.seen1 = (to + shift) >> 1;
      *work = w;
      if (w.ctx > sv.max_pages * PAGE) atomicOr(args.errors, (uint32_t)ffb::ERR_KV4_PAGE);
    }
  };
  // Each role has a loop of its own, so that the registers of one are not those of another.
  auto for_items = [&](auto&& before, auto&& role) {
    for (int step = 0;; ++step) {
      before(step);
      __syncthreads();
      if (work->kvh < 0) break;
      const bool two = work->clast >= work->c0 + 128;
      const int nblk = work->blocks();
      role(two, nblk);
      if (!__syncthreads_and(!*abort_flag)) break;  // all roles, or none
      blk0 += nblk;
      tiles += nblk > 0;
      if (two) {
        blkB0 += nblk;
        tilesB += nblk > 0;
      }
    }
  };
  auto nothing = [](int) {};

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_ISSUE));
    for_items([&](int step) { if (warp == 0) find_work(step); }, [&](const bool two, const int nblk) {
    if (warp == 0) {
      // ---------------------------------------------------------------- raw pages
      if (lane == 0) {
        const Work w = *work;
        int bad_pair = 0;
        for (int i = 0; i < 2 * nblk; ++i) {
          const uint32_t u = 2 * blk0 + i, s = u % RAW;
          if (u >= RAW && !wait_held(&raw_empty[s], ((u / RAW) & 1u) ^ 1u, abort_flag)) {
            *abort_flag = 1;
            break;
          }
          int page = -1;
          if (w.i0 + i < w.i1) {
            page = __ldg(w.table + w.page_index(w.i0 + i));
            if (page < 0 || page >= sv.num_pages) {
              atomicOr(args.errors, (uint32_t)ffb::ERR_KV4_PAGE);
              page = -1;
            }
          }
          raw_bad[s] = page < 0;
          bad_pair = (i & 1) ? bad_pair | (page < 0 ? 2 : 0) : (page < 0 ? 1 : 0);
          if (i & 1) blk_bad[(blk0 + (i >> 1)) & 15] = bad_pair;
          if (page >= 0) {
            mbar_arrive_expect_tx(&raw_full[s], RECORD);
            bulk_load(raw + s * RECORD, sv.pages + ((int64_t)page * sv.HK + w.kvh) * RECORD, RECORD, &raw_full[s]);
          } else {
            mbar_arrive(&raw_full[s]);
          }
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMAs
      // The whole warp walks the blocks and one elected thread issues, so that descriptors and
      // addresses stay in uniform registers: issued by one diverged thread an MMA took 130 clocks
      // whatever its size.
      constexpr uint32_t idesc_s = idesc_bf16(128, 128);
      constexpr uint32_t idesc_o = idesc_bf16(128, 128) | (1u << 16);  // B (= V) MN-major
      const uint32_t qbase = smem_u32(sq), kvbase = smem_u32(slots);
      const bool leader = elect_one();
      auto wait_uniform = [&](uint64_t* bar, uint32_t parity) {
        const bool done = __all_sync(0xffffffffu, wait_held(bar, parity, abort_flag)) != 0;
        tc_fence_after();
        return done;
      };
      auto wait_slot = [&](uint32_t u) { return wait_uniform(&slot_full[u % SLOTS], (u / SLOTS) & 1u); };
      auto scores = [&](int x, uint32_t u, bool free_slot) {
        const uint64_t qd = umma_desc_sw128(qbase + x * TILE), kd = umma_desc_sw128(kvbase + (u % SLOTS) * TILE);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_f16(128 * x, qd + ((kk >> 2) * HALF + (kk & 3) * 32) / 16, kd + ((kk >> 2) * HALF + (kk & 3) * 32) / 16, idesc_s,
                     kk > 0 ? 1u : 0u);
          umma_commit(&s_full[x]);
          if (free_slot) umma_commit(&slot_empty[u % SLOTS]);
        }
        __syncwarp();
      };
      // O += P V, a page's keys as soon as their probabilities are there
      auto product = [&](int x, uint32_t u, uint32_t parity, bool first, bool free_slot) {
        const uint64_t vd = umma_desc_sw128_mn(kvbase + (u % SLOTS) * TILE, HALF);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!wait_uniform(&p_full[2 * x + half], parity)) return false;
          if (leader) {
#pragma unroll
            for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
              umma_f16_ts(256 + 128 * x, 128 * x + 8 * kk, vd + kk * 2048 / 16, idesc_o, (!first || kk > 0) ? 1u : 0u);
            if (half) {
              umma_commit(&o_done[x]);
              if (free_slot) umma_commit(&slot_empty[u % SLOTS]);
            }
          }
          __syncwarp();
        }
        return true;
      };
      bool go = true;
      if (nblk > 0) {
        go = wait_uniform(&q_full[0], tiles & 1u) && (!two || wait_uniform(&q_full[1], tilesB & 1u)) && wait_slot(2 * blk0);
        if (go) {
          scores(0, 2 * blk0, !two);
          if (two) scores(1, 2 * blk0, true);
        }
      }
      for (int j = 0; j < nblk && go; ++j) {
        const uint32_t uv = 2 * (blk0 + j) + 1, uk = uv + 1;
        const bool more = j + 1 < nblk;
        go = wait_slot(uv) && product(0, uv, (blk0 + j) & 1u, j == 0, !two);
        if (!go) break;
        if (more) {
          go = wait_slot(uk);
          if (!go) break;
          scores(0, uk, !two);
        }
        if (two) {
          go = product(1, uv, (blkB0 + j) & 1u, j == 0, true);
          if (!go) break;
          if (more) scores(1, uk, true);
        }
      }
      if (!go) *abort_flag = 1;
    }
    });
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_DEQUANT));
    for_items(nothing, [&](const bool, const int nblk) {
      // ---------------------------------------------------------------- dequantisation
      const int r8 = 8 * (warp - 12);  // this warp's eight tokens of a page
      // K: token pairs (r, r ^ 5) x four chunks meet all banks on the load and on the store;
      // V: tokens {0, 1, 6, 7} / {2, 3, 4, 5} of eight x two neighbouring 16-byte pairs
      const int kt = lane & 3, kr = r8 + ((lane >> 3) ^ ((lane & 4) ? 5 : 0));
      const int vk = (lane >> 1) & 3, pair = 2 * (lane >> 4) + (lane & 1);
      const int vr = r8 + ((lane & 8) ? 2 + vk : (vk < 2 ? vk : 4 + vk));
      const Work w = *work;
      for (int j = 0; j < nblk && ok; ++j) {
        const uint32_t u = 2 * (blk0 + j);  // the K tile's number, and the first page's
        // tokens past the newest row's position are held by nobody: whatever is there is not used
        int live[2];
        bool got = true;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          got = got && wait_held(&raw_full[(u + a) % RAW], ((u + a) / RAW) & 1u, abort_flag);
          const int i = w.i0 + 2 * j + a, key0 = i < w.i1 ? w.page_index(i) * PAGE : 0;
          live[a] = raw_bad[(u + a) % RAW] ? 0 : min(max(w.ps.kend - key0, 0), PAGE);
        }
#pragma unroll
        for (int is_v = 0; is_v < 2; ++is_v) {
          const uint32_t slot = (u + is_v) % SLOTS;
          got = got && (u + is_v < SLOTS || wait_held(&slot_empty[slot], (((u + is_v) / SLOTS) & 1u) ^ 1u, abort_flag));
          got = __all_sync(0xffffffffu, got);  // one verdict for the warp
          if (!got) break;
          uint8_t* dst = slots + slot * TILE;
          // both pages' loads first: one after the other their latencies bound the whole kernel
          uint4 c[2];
          uint2 sc[2];
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const uint8_t* rec = raw + ((u + a) % RAW) * RECORD;
            c[a] = make_uint4(0u, 0u, 0u, 0u);
            sc[a] = make_uint2(0u, 0u);
            if (!is_v && kr < live[a]) {
              c[a] = *reinterpret_cast<const uint4*>(rec + 64 * kr + 16 * kt);
              sc[a] = *reinterpret_cast<const uint2*>(rec + K_SCALES + 8 * kr);
              const uint2 vs = *reinterpret_cast<const uint2*>(rec + V_SCALES + 8 * kr);
              if (not_finite2(vs.x) || not_finite2(vs.y)) sc[a] = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
            }
            if (is_v && vr < live[a]) {
              c[a] = *reinterpret_cast<const uint4*>(rec + V_CODES + 64 * vr + 16 * (pair ^ ((vr & 4) >> 1)));
              sc[a] = *reinterpret_cast<const uint2*>(rec + V_SCALES + 8 * vr);
              if (not_finite2(sc[a].x) || not_finite2(sc[a].y)) sc[a] = make_uint2(0u, 0u);
            }
          }
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const uint32_t words[4] = {c[a].x, c[a].y, c[a].z, c[a].w};
            if (!is_v) {
              const uint32_t scale[4] = {__byte_perm(sc[a].x, 0, 0x1010), __byte_perm(sc[a].x, 0, 0x3232),
                                         __byte_perm(sc[a].y, 0, 0x1010), __byte_perm(sc[a].y, 0, 0x3232)};
              uint8_t* row = dst + (64 * a + kr) * 128;
#pragma unroll
              for (int q = 0; q < 4; ++q)
                *reinterpret_cast<uint4*>(row + (q >> 1) * HALF + (((4 * (q & 1) + kt) ^ (kr & 7)) << 4)) =
                    dequant8(words[q], scale[q]);
            } else {  // chunks 2 pair, 2 pair + 1 of V, two words each
              uint8_t* row = dst + (pair >> 1) * HALF + (64 * a + vr) * 128;
#pragma unroll
              for (int q = 0; q < 4; ++q)
                *reinterpret_cast<uint4*>(row + (((4 * (pair & 1) + q) ^ (vr & 7)) << 4)) =
                    dequant8(words[q], (q & 1) ? sc[a].y : sc[a].x);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&slot_full[slot]);
            if (is_v) {
              mbar_arrive(&raw_empty[u % RAW]);
              mbar_arrive(&raw_empty[(u + 1) % RAW]);
            }
          }
        }
        if (!got) {
          ok = false;
          *abort_flag = 1;
        }
      }
    });
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    for_items(nothing, [&](const bool two, const int nblk) {
      // ---------------------------------------------------------------- softmax
      const int x = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
      if (x == 0 || two) {
        const uint32_t base_blk = x ? blkB0 : blk0;
        const volatile Work& w = *work;
        const float base = fmaxf(fabsf(args.scale_log2), 1e-37f);  // scale 0: a masked -inf stays one
        float sc = base;                                           // smaller while the row's scores are vast
        // this thread's column (past the last: the last one's), and its row and head, which shuffles
        // hand on
        auto column = [&] { return min(w.c0 + 128 * x + r, w.clast); };
        auto place_of = [&] { return w.r0 + column() / G; };
        auto head_of = [&] { return w.kvh * G + column() % G; };
        // this warp's 32 rows of Q, negated for a negative scale (exact), eight channels a chunk in
        // the order 0 4 1 5 2 6 3 7; sixteen lanes copy one row, eight loads in flight.  A tile without
        // blocks has no queries: no product would keep its warps from staging output over rows that
        // others still write
        if (nblk > 0) {
          const uint32_t flip = args.scale_log2 < 0.f ? 0x80008000u : 0u;
          const int ch = lane & 15, place = place_of(), head = head_of();
#pragma unroll
          for (int k0 = 0; k0 < 32; k0 += 16) {
            uint4 in[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int from = k0 + 2 * k + (lane >> 4);
              const int64_t at = (int64_t)__shfl_sync(0xffffffffu, head, from) * sv.T + __shfl_sync(0xffffffffu, place, from);
              in[k] = __ldg(reinterpret_cast<const uint4*>(args.q + at * D + 8 * ch));
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int rr = quarter * 32 + k0 + 2 * k + (lane >> 4);
              const uint4 v = w.c0 + 128 * x + rr <= w.clast ? in[k] : make_uint4(0u, 0u, 0u, 0u);
              // channels 8 ch .. of group ch / 4: chunk 4 (j & 1) + t of half j / 2 with j = ch / 4, t = ch % 4
              const uint4 y = make_uint4(__byte_perm(v.x, v.z, 0x5410) ^ flip, __byte_perm(v.x, v.z, 0x7632) ^ flip,
                                         __byte_perm(v.y, v.w, 0x5410) ^ flip, __byte_perm(v.y, v.w, 0x7632) ^ flip);
              *reinterpret_cast<uint4*>(sq + x * TILE + (ch >> 3) * HALF + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4)) = y;
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[x]);
        }
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        const uint32_t st = tmem + lane_addr + 128 * x, ot = tmem + lane_addr + 256 + 128 * x;
        float m = -INFINITY, neg = 0.f, l = 0.f;  // neg: -m, 0 while nothing has been seen
        for (int j = 0; j < nblk; ++j) {
          const bool part = j < w.seen0 || j >= w.seen1;
          if (!__all_sync(0xffffffffu, wait_held(&s_full[x], (base_blk + j) & 1u, abort_flag) && !*abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int bad = blk_bad[(blk0 + j) & 15];
          if (part || bad) {  // rare blocks: the scores that do not count become -inf where they lie
            const int ia = w.i0 + 2 * j;
            int key0[2];
#pragma unroll
            for (int a = 0; a < 2; ++a)
              key0[a] = (ia + a < w.ps.n_sink ? ia + a : w.ps.first_page + ia + a - w.ps.n_sink) * PAGE;
            // the keys of a page that this column sees: c <= hi and (c >= lo or c < sk)
            const int pos = w.first_pos + column() / G;
            const int top = min(pos, w.ps.kend - 1), low = args.window > 0 ? pos - args.window + 1 : 0;
            const int hi[2] = {(bad & 1) ? -1 : top - key0[0], (bad & 2) ? -1 : top - key0[1]};
            const int lo[2] = {low - key0[0], low - key0[1]}, sk[2] = {args.sinks - key0[0], args.sinks - key0[1]};
#pragma unroll 1
            for (int q = 0; q < 8; ++q) {
              const int first = 16 * (q & 3), h = hi[q >> 2] - first, l0 = lo[q >> 2] - first, s0 = sk[q >> 2] - first;
              uint32_t y[16];
              tmem_ld16_async(st + 16 * q, y);
              tmem_wait_ld();
              reg_fence(y);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (!(e <= h && (e >= l0 || e < s0))) y[e] = 0xff800000u;
              tmem_st16(st + 16 * q, y);
            }
            tmem_wait_st();
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          uint32_t v[2][16];
          tmem_ld16_async(st, v[0]);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            tmem_wait_ld();
            reg_fence(v[q & 1]);
            if (q < 7) tmem_ld16_async(st + 16 * (q + 1), v[(q + 1) & 1]);
#pragma unroll
            for (int e = 0; e < 16; e += 2)
              mx[(e >> 1) & 3] = fmaxf(mx[(e >> 1) & 3], fmaxf(__uint_as_float(v[q & 1][e]), __uint_as_float(v[q & 1][e + 1])));
          }
          uint32_t w[2][16];  // the scores again, for the probabilities: on their way while the maximum is looked at
          tmem_ld16_async(st, w[0]);
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const bool grow = top * sc > m + LAZY;
          if (__any_sync(0xffffffffu, grow)) {
            const float to_sc = grow ? base * vast_scale(top * base) : sc, nm = grow ? top * to_sc : m;
            const float alpha = grow ? (to_sc == sc ? ex2(m - nm) : 0.f) : 1.f;
            sc = to_sc;
            l *= alpha;
            m = nm;
            neg = m == -INFINITY ? 0.f : -m;
            if (j > 0) {
              if (!__all_sync(0xffffffffu, wait_held(&o_done[x], (base_blk + j - 1) & 1u, abort_flag))) {
                ok = false;
                break;
              }
              tc_fence_after();
#pragma unroll 1
              for (int q = 0; q < 8; ++q) {
                uint32_t y[16];
                tmem_ld16_async(ot + 16 * q, y);
                tmem_wait_ld();
                reg_fence(y);
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * alpha);
                tmem_st16(ot + 16 * q, y);
              }
              tmem_wait_st();
            }
          }
          const float2 neg2 = make_float2(neg, neg), sc2 = make_float2(sc, sc);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uint32_t p[8];
            tmem_wait_ld();
            reg_fence(w[q & 1]);
            if (q < 7) tmem_ld16_async(st + 16 * (q + 1), w[(q + 1) & 1]);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float2 y = fma2(make_float2(__uint_as_float(w[q & 1][e]), __uint_as_float(w[q & 1][e + 1])), sc2, neg2);
              const float2 z = make_float2(ex2(y.x), ex2(y.y));
              sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], z);
              p[e >> 1] = pack_bf16(z.x, z.y);
            }
            tmem_st8(st + 8 * q, p);
            if (q == 3 || q == 7) {  // a page is done: its product may start
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_full[2 * x + (q >> 2)]);
            }
          }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        }
        if (ok && nblk > 0)
          ok = __all_sync(0xffffffffu, wait_held(&o_done[x], (base_blk + nblk - 1) & 1u, abort_flag) && !*abort_flag);
        if (!ok) *abort_flag = 1;
        if (ok) {
          tc_fence_after();
          if (w.parts > 1) {
            // fp32 sums in the columns' order, four columns of all 256 rows next to each other, so that a
            // warp stores 512 bytes in a row; kv4_join_tc_kernel takes them back to channels
            const int64_t part = (int64_t)blockIdx.x - args.whole;
            const int column = 128 * x + r;
            const bool live_row = w.c0 + column <= w.clast;
            float4* to = reinterpret_cast<float4*>(args.part_o) + part * (256 * D / 4) + column;
            if (live_row)
              *reinterpret_cast<float2*>(args.part_ml + (part * 256 + column) * 2) = make_float2(sc == base ? m : m * (base / sc), l);
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              uint32_t v[32];
              if (nblk > 0) {
                tmem_ld32_async(ot + 32 * q, v);
                tmem_wait_ld();
                reg_fence(v);
              } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = 0u;
              }
              if (live_row)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  to[256 * (8 * q + e)] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]),
                                                      __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
            }
          } else {
            // rows staged over this warp's part of the Q tile (every S product has been read), words
            // of two channels at word ^ (row % 32); 32 columns hold the channel pair 2 q of each 8
            const float rl = l == 0.f ? 0.f : 1.f / l;
            uint32_t* stage = reinterpret_cast<uint32_t*>(sq + x * TILE) + r * 64;
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              uint32_t v[32];
              if (nblk > 0) {
                tmem_ld32_async(ot + 32 * q, v);
                tmem_wait_ld();
                reg_fence(v);
              } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = 0u;
              }
#pragma unroll
              for (int e = 0; e < 16; ++e) {  // chunk 4 q (+ half) and 4 q + 2 (+ half): chunks g = 2 q and 2 q + 1 of V
                const int half = e >> 3, d8 = 8 * half + nibble_of(e & 7);  // channels 8 d8 + 2 q, + 1
                stage[(4 * d8 + q) ^ lane] = pack_bf16(__uint_as_float(v[e]) * rl, __uint_as_float(v[16 + e]) * rl);
              }
            }
            __syncwarp();
            const uint32_t* src = reinterpret_cast<const uint32_t*>(sq + x * TILE) + quarter * 32 * 64;
            const int place = place_of(), head = head_of(), n = min(w.clast - (w.c0 + 128 * x + quarter * 32) + 1, 32);
#pragma unroll 8
            for (int k = 0; k < n; ++k) {
              uint32_t* dst = reinterpret_cast<uint32_t*>(args.out) +
                              ((int64_t)__shfl_sync(0xffffffffu, place, k) * args.HQ + __shfl_sync(0xffffffffu, head, k)) * 64;
              dst[lane] = src[64 * k + (lane ^ k)];
              dst[32 + lane] = src[64 * k + 32 + (lane ^ k)];
            }
            __syncwarp();
          }
          tc_fence_before();
        }
      }
    });
  }

  if (warp == 1) {
    // every MMA issued has completed before tensor and shared memory are released (the thread that
    // elect_one names is the same every time)
    if (elect_one()) {
      volatile int never = 0;
      umma_commit(last);
      mbar_wait_bounded(last, 0, &never, 200000000ull);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) {  // some role gave up (which the roles' last barrier has settled)
    atomicOr(args.errors, (uint32_t)ffb::ERR_ATTN_TIMEOUT);
    // pages in flight land before the CTA leaves: the producer may have ended before the others gave up
    volatile int never = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < 2 * RAW; ++i) mbar_wait_bounded(&raw_full[i >> 1], i & 1u, &never, 20000000ull);
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

namespace kv4 {
cudaError_t launch_attention_tc(const AttnArgs& a, unsigned ctas, cudaStream_t stream) {
  // setmaxnreg is right for one number of registers at the launch alone
  static const int launch_regs = [] {
    cudaFuncAttributes f;
    return cudaFuncGetAttributes(&f, kv4_attention_tc_kernel) == cudaSuccess ? f.numRegs : 0;
  }();
  if (launch_regs != LAUNCH_REGS) return cudaErrorInvalidKernelImage;
  cudaError_t e = ffb::set_smem_attr(reinterpret_cast<const void*>(kv4_attention_tc_kernel), SMEM);
  if (e == cudaSuccess)
    e = ffb::launch(kv4_attention_tc_kernel, dim3(ctas), dim3(THREADS), SMEM, stream, a);
  return e;
}
}  // namespace kv4
