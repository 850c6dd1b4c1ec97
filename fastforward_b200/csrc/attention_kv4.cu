// Attention over the 4-bit paged K/V cache (layout: kv4.cuh) for few query rows a sequence:
// single-token decoding and short runs of new tokens.
//
//   o[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - m),  x_j = scale log2(e) q.k_j
// over the keys j <= the row's position, inside the window or among the first `sinks`.
//
// The floor is the bytes of the visible pages (144 a token and K/V head), so the kernel is
// built to keep bulk copies in flight and to spend few instructions a byte:
//   - one CTA takes one (sequence, K/V head, 8 NT query columns, share of the pages): the
//     columns are the (row, head of the group) pairs, so a page is read once for all the
//     query heads that share it.  16 warps in four groups; a group has its own ring of
//     STAGES page records, filled by cp.async.bulk, and its four warps take 16 tokens each;
//   - the products run on mma.sync m16n8k16 with the tokens on M and the query columns on N
//     (S^T = K Q^T, O^T = V^T P^T): with G <= 8 heads a group a tcgen05 tile of 128 rows
//     would be nearly empty, and its operands would have to be written to shared memory as
//     bf16, four times the bytes of the codes.  Here a code becomes bf16 in a register:
//     0x4300 | nibble is 128 + nibble;
//   - K: the offset 136 of every operand is taken out by starting each group's accumulator at
//     -136 sum(q) of the group's channels; the group's scale multiplies the fp32 sums;
//   - V: the offset is subtracted (exact), the scale multiplies the probability before its
//     one rounding to bf16, once per group of channels; P^T is formed by movmatrix;
//   - the running maximum moves only when a score passes it by more than 8 (in base 2), which
//     a vote finds: p <= 2^8, nothing overflows, and the rescaling is rare.
// S, the maxima, the sums and O are fp32; P (times V's scale) is rounded to bf16, the type of
// the tensor core's operand, with relative error 2^-9 of each term.
// Shares of a long axis are joined by kv4_combine_kernel (fp32 partials in the workspace).
#include "kv4.cuh"
#include "pdl.cuh"

#include <math.h>
#include <type_traits>

namespace {

using namespace kv4;

constexpr int GROUPS = 4;             // page streams of a CTA
constexpr int GW = 2;                 // warps of a group; each takes PAGE / GW tokens of a page
constexpr int WARPS = GROUPS * GW;
constexpr int THREADS = 32 * WARPS;
constexpr int CS = D + 4;             // fp32 pitch of a column in the final exchange (spreads the banks)
constexpr float LAZY = 8.f;

template <int NT>
struct Shape {
  // two CTAs an SM, so that one starts or ends while the other streams; 16 columns need the
  // registers (64 sums a thread) and the stages of one
  static constexpr int PER_SM = NT == 1 ? 2 : 1;
  static constexpr int STAGES = NT == 1 ? 3 : 5;  // page records in flight per group
  static constexpr int RING = GROUPS * STAGES * RECORD;
  static constexpr int BARS = 2 * GROUPS * STAGES * 8 + GROUPS * STAGES * 4 + 16;
  // ring | Q fragments [NT][4][32] uint4 | offsets [NT][2][32] float4 | barriers
  static constexpr int SMEM = RING + NT * 4 * 512 + NT * 2 * 512 + BARS + 128;
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// The token of fragment row r (0..7): 2 <-> 3 and 6 <-> 7 trade places, so that the eight lanes
// of a load phase meet rows of both parities and, with V's exchanged halves, all banks.
__device__ __forceinline__ int token_of(int r) { return r ^ ((r >> 1) & 1); }

template <int NT>
__global__ void __launch_bounds__(THREADS, Shape<NT>::PER_SM) kv4_attention_kernel(const AttnArgs args) {
  constexpr int QT = 8 * NT, STAGES = Shape<NT>::STAGES, RING = Shape<NT>::RING;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  uint4* sq = reinterpret_cast<uint4*>(smem + RING);                     // [NT][4][32]
  float4* soff = reinterpret_cast<float4*>(smem + RING + NT * 4 * 512);  // [NT][2][32]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + RING + NT * 6 * 512);
  uint64_t* empty = full + GROUPS * STAGES;
  int* bad = reinterpret_cast<int*>(empty + GROUPS * STAGES);  // per stage: the page id was outside the cache
  volatile int* abort_flag = bad + GROUPS * STAGES;

  const Seqs& sq_ = args.seqs;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = warp / GW, gw = warp % GW, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % args.splits;
  const int kvh = (blockIdx.x / args.splits) % sq_.HK, b = blockIdx.x / (args.splits * sq_.HK);
  const int G = args.HQ / sq_.HK;
  const bool producer = gw == 0 && lane == 0;

  if (tid == 0) {
    for (int i = 0; i < GROUPS * STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], GW);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  if (tid == 0) pdl_launch();

  const int r0 = min(max(__ldg(sq_.row_start + b), 0), sq_.T);
  const int r1 = min(max(__ldg(sq_.row_start + b + 1), r0), sq_.T);
  const int S = r1 - r0, ctx = max(__ldg(sq_.ctx_len + b), 0);
  const int ncols = S * G;
  const int* table = sq_.table + b * sq_.table_stride;
  // The group's ring: the stage and phase parity of its next page to use; `fill` of the next to load.
  int use = 0, fill = 0, freed = 0;
  uint32_t use_ph = 0, freed_ph = 0;
  uint64_t* gfull = full + group * STAGES;
  uint64_t* gempty = empty + group * STAGES;
  uint8_t* gring = smem + group * STAGES * RECORD;
  if (ctx > sq_.max_pages * PAGE && S > 0 && tid == 0) atomicOr(&ffb_device_error_word, (uint32_t)ffb::ERR_KV4_PAGE);

  for (int c0 = (int)blockIdx.y * QT; c0 < ncols; c0 += (int)gridDim.y * QT) {
    const int clast = min(c0 + QT, ncols) - 1;
    const int pos_lo = ctx - S + c0 / G, pos_hi = ctx - S + clast / G;
    const PageSet ps = pages_of(pos_lo, pos_hi, sq_.max_pages, args.window, args.sinks);
    const int i0 = (int)((int64_t)split * ps.n / args.splits), i1 = (int)((int64_t)(split + 1) * ps.n / args.splits);
    const int cnt = max(0, (i1 - i0 - group + GROUPS - 1) / GROUPS);  // pages i0 + group + GROUPS k of this group
    // page indexes [whole_lo, whole_hi) are seen in full by every column
    const int whole_key = args.window > 0 ? max(0, pos_hi - args.window + 1) : 0;
    const int whole_lo = ps.n_sink + max(0, (whole_key + PAGE - 1) / PAGE - ps.first_page);
    const int whole_hi = ps.n_sink + min(max(pos_lo + 1, 0), ps.kend) / PAGE - ps.first_page;
    auto page_index = [&](int i) { return i < ps.n_sink ? i : ps.first_page + i - ps.n_sink; };
    auto issue = [&](int k) {  // the producer lane
      const int page = __ldg(table + page_index(i0 + group + GROUPS * k));
      const bool ok = page >= 0 && page < sq_.num_pages;
      bad[group * STAGES + fill] = !ok;
      if (ok) {
        mbar_arrive_expect_tx(&gfull[fill], RECORD);
        bulk_load(gring + fill * RECORD, sq_.pages + ((int64_t)page * sq_.HK + kvh) * RECORD, RECORD, &gfull[fill]);
      } else {
        atomicOr(&ffb_device_error_word, (uint32_t)ffb::ERR_KV4_PAGE);
        mbar_arrive(&gfull[fill]);
      }
      fill = fill + 1 == STAGES ? 0 : fill + 1;
    };
    // the stage of the oldest page not known to be free: waits until its warps are done with it
    auto reclaim = [&]() {
      const bool done = mbar_wait_bounded(&gempty[freed], freed_ph, abort_flag);
      if (++freed == STAGES) {
        freed = 0;
        freed_ph ^= 1u;
      }
      return done;
    };
    int issued = 0, reclaimed = 0;
    if (producer)
      for (; issued < min(cnt, STAGES); ++issued) issue(issued);

    // query fragments of this tile, once per CTA: lane (g, t) of column tile n holds channels
    // 32 j + 8 t .. + 7 of column 8 n + g as the pairs (e, e + 4) that pair136 gives
    for (int f = warp; f < 4 * NT; f += WARPS) {
      const int n = f >> 2, j = f & 3;
      const int c = c0 + 8 * n + g;
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (c <= clast) {
        const int row = r0 + c / G, h = kvh * G + c % G;
        x = __ldg(reinterpret_cast<const uint4*>(args.q + ((int64_t)h * sq_.T + row) * D + 32 * j + 8 * t));
      }
      float sum = lo_of(x.x) + hi_of(x.x) + lo_of(x.y) + hi_of(x.y) + lo_of(x.z) + hi_of(x.z) + lo_of(x.w) + hi_of(x.w);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sq[(n * 4 + j) * 32 + lane] = make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632),
                                               __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
      // lane (g', t') of the score fragment needs the sums of columns 2 t' and 2 t' + 1
      const float s0 = __shfl_sync(0xffffffffu, sum, 8 * t), s1 = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      float2* dst = reinterpret_cast<float2*>(soff) + ((n * 2 + (j >> 1)) * 32 + lane) * 2 + (j & 1);
      *dst = make_float2(-136.f * s0, -136.f * s1);
    }
    __syncthreads();

    uint32_t qf[NT == 1 ? 16 : 1];
    float off[NT == 1 ? 8 : 1];
    if constexpr (NT == 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 x = sq[j * 32 + lane];
        qf[4 * j] = x.x; qf[4 * j + 1] = x.y; qf[4 * j + 2] = x.z; qf[4 * j + 3] = x.w;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 x = soff[j * 32 + lane];
        off[4 * j] = x.x; off[4 * j + 1] = x.y; off[4 * j + 2] = x.z; off[4 * j + 3] = x.w;
      }
    }

    float o[8][NT][4], m[2 * NT], l[2 * NT];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
    int pos[2 * NT];  // positions of this lane's columns
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
      const int c = c0 + 8 * (i >> 1) + 2 * t + (i & 1);
      pos[i] = c <= clast ? ctx - S + c / G : -1;
    }

    // sixteen tokens of one page, from tok0 on; MASKED: some column may not see some of them
    auto tile = [&](const uint8_t* rec, int tok0, int key0, auto masked_tag) {
      constexpr bool MASKED = decltype(masked_tag)::value;
      const int ra = tok0 + token_of(g), rb = ra + 8;  // tokens of fragment rows g and g + 8
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
      {
        const uint4 ka = *reinterpret_cast<const uint4*>(rec + 64 * ra + 16 * t);
        const uint4 kb = *reinterpret_cast<const uint4*>(rec + 64 * rb + 16 * t);
        const uint2 sa = *reinterpret_cast<const uint2*>(rec + K_SCALES + 8 * ra);
        const uint2 sb = *reinterpret_cast<const uint2*>(rec + K_SCALES + 8 * rb);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
        const float fa[4] = {lo_of(sa.x), hi_of(sa.x), lo_of(sa.y), hi_of(sa.y)};
        const float fb[4] = {lo_of(sb.x), hi_of(sb.x), lo_of(sb.y), hi_of(sb.y)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a0 = pair136(wa[j], 0), a1 = pair136(wb[j], 0), a2 = pair136(wa[j], 1), a3 = pair136(wb[j], 1);
          const uint32_t a4 = pair136(wa[j], 2), a5 = pair136(wb[j], 2), a6 = pair136(wa[j], 3), a7 = pair136(wb[j], 3);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint32_t q0, q1, q2, q3;
            float c[4] = {0.f, 0.f, 0.f, 0.f}, d0, d1;
            if constexpr (NT == 1) {
              q0 = qf[4 * j]; q1 = qf[4 * j + 1]; q2 = qf[4 * j + 2]; q3 = qf[4 * j + 3];
              d0 = off[2 * j]; d1 = off[2 * j + 1];
            } else {
              const uint4 x = sq[(n * 4 + j) * 32 + lane];
              q0 = x.x; q1 = x.y; q2 = x.z; q3 = x.w;
              const float2 y = reinterpret_cast<const float2*>(soff)[((n * 2 + (j >> 1)) * 32 + lane) * 2 + (j & 1)];
              d0 = y.x; d1 = y.y;
            }
            mma16816(c, a0, a1, a2, a3, q0, q1);
            mma16816(c, a4, a5, a6, a7, q2, q3);
            s[n][0] = fmaf(c[0] + d0, fa[j], s[n][0]);
            s[n][1] = fmaf(c[1] + d1, fa[j], s[n][1]);
            s[n][2] = fmaf(c[2] + d0, fb[j], s[n][2]);
            s[n][3] = fmaf(c[3] + d1, fb[j], s[n][3]);
          }
        }
      }
      bool grow = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[n][e] * args.scale_log2;
          if constexpr (MASKED) {
            const int key = key0 + (e < 2 ? ra : rb), p = pos[2 * n + (e & 1)];
            if (key > p || key >= ps.kend || (args.window > 0 && p - key >= args.window && key >= args.sinks)) x = -INFINITY;
          }
          s[n][e] = x;
          grow |= x > m[2 * n + (e & 1)] + LAZY;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
          float x = fmaxf(s[i >> 1][i & 1], s[i >> 1][2 + (i & 1)]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float nm = fmaxf(m[i], x);
          const float a = nm == -INFINITY ? 1.f : ex2(m[i] - nm);  // nothing seen yet: keep zeros
          m[i] = nm;
          l[i] *= a;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            o[d][i >> 1][i & 1] *= a;
            o[d][i >> 1][2 + (i & 1)] *= a;
          }
        }
      }
      uint32_t pb[NT][8];  // P^T fragments, V's scale of group j folded in
      {
        const uint2 sa = *reinterpret_cast<const uint2*>(rec + V_SCALES + 8 * ra);
        const uint2 sb = *reinterpret_cast<const uint2*>(rec + V_SCALES + 8 * rb);
        const float fa[4] = {lo_of(sa.x), hi_of(sa.x), lo_of(sa.y), hi_of(sa.y)};
        const float fb[4] = {lo_of(sb.x), hi_of(sb.x), lo_of(sb.y), hi_of(sb.y)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // a masked score stays 0 even while the maximum is still -inf
            p[e] = MASKED && s[n][e] == -INFINITY ? 0.f : ex2(s[n][e] - m[2 * n + (e & 1)]);
            l[2 * n + (e & 1)] += p[e];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float y[4] = {p[0] * fa[j], p[1] * fa[j], p[2] * fb[j], p[3] * fb[j]};
            if constexpr (MASKED) {  // nothing of a masked token counts, whatever its scale holds
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (p[e] == 0.f) y[e] = 0.f;
            }
            pb[n][2 * j] = transpose8x8(pack_bf16(y[0], y[1]));
            pb[n][2 * j + 1] = transpose8x8(pack_bf16(y[2], y[3]));
          }
        }
      }
      // V^T fragments: columns 2t, 2t+1, 2t+8, 2t+9 of the MMA are these four tokens
      const int ta = tok0 + token_of(2 * t), tb = tok0 + token_of(2 * t + 1);
      const uint8_t* v = rec + V_CODES + 8 * (g ^ (4 * (t >> 1)));
      const uint2 v0 = *reinterpret_cast<const uint2*>(v + 64 * ta), v1 = *reinterpret_cast<const uint2*>(v + 64 * tb);
      const uint2 v2 = *reinterpret_cast<const uint2*>(v + 64 * ta + 512), v3 = *reinterpret_cast<const uint2*>(v + 64 * tb + 512);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t x0 = half ? v0.y : v0.x, x1 = half ? v1.y : v1.x, x2 = half ? v2.y : v2.x, x3 = half ? v3.y : v3.x;
#pragma unroll
        for (int quart = 0; quart < 2; ++quart) {
          const uint32_t sel = quart ? 0x7632 : 0x5410;
          const uint32_t lo = __byte_perm(x0, x1, sel), hi = __byte_perm(x2, x3, sel);  // tokens (2t, 2t+1), (2t+8, 2t+9)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int mt = 4 * half + 2 * quart + u;  // channels 16 mt + g and 16 mt + 8 + g
            const uint32_t a0 = minus136(pair136(lo, 2 * u)), a1 = minus136(pair136(lo, 2 * u + 1));
            const uint32_t a2 = minus136(pair136(hi, 2 * u)), a3 = minus136(pair136(hi, 2 * u + 1));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(o[mt][n], a0, a1, a2, a3, pb[n][2 * (mt >> 1)], pb[n][2 * (mt >> 1) + 1]);
          }
        }
      }
    };

    bool ok = true;
    for (int k = 0; k < cnt; ++k) {
      // one verdict for the warp: its lanes stay together whatever each of them saw
      if (!__all_sync(0xffffffffu, mbar_try_wait(&gfull[use], use_ph)) &&
          !__all_sync(0xffffffffu, mbar_wait_bounded(&gfull[use], use_ph, abort_flag))) {
        ok = false;
        break;
      }
      const int i = i0 + group + GROUPS * k;
      if (!bad[group * STAGES + use]) {
        const uint8_t* rec = gring + use * RECORD;
        constexpr int TOK = PAGE / GW;
        if (i >= whole_lo && i < whole_hi) {
#pragma unroll 1
          for (int a = 0; a < TOK; a += 16) tile(rec, TOK * gw + a, 0, std::integral_constant<bool, false>{});
        } else {
          const int key0 = page_index(i) * PAGE;
#pragma unroll 1
          for (int a = 0; a < TOK; a += 16)
            if (key0 + TOK * gw + a < ps.kend) tile(rec, TOK * gw + a, key0, std::integral_constant<bool, true>{});
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&gempty[use]);
      if (++use == STAGES) {
        use = 0;
        use_ph ^= 1u;
      }
      // refill the stage of the page before this one (the group's warps are about to be done with it)
      if (producer && k > 0 && issued < cnt) {
        if (reclaim()) issue(issued++);
        else *abort_flag = 1;  // the waits for the pages never issued give up on it
        ++reclaimed;
      }
    }
    if (!ok) *abort_flag = 1;
    if (producer) {
      volatile int never = 0;
      if (*abort_flag) {  // copies in flight must land before the CTA leaves
        for (int i = 0; i < STAGES; ++i) {
          mbar_wait_bounded(&gfull[i], 0, &never, 20000000ull);
          mbar_wait_bounded(&gfull[i], 1, &never, 20000000ull);
        }
      } else {  // every stage free again: the ring is used for the exchange, then for the next tile
        for (; reclaimed < cnt; ++reclaimed)
          if (!reclaim()) *abort_flag = 1;
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
    }
    __syncthreads();  // all pages consumed: the ring becomes the exchange buffer
    if (*abort_flag) break;  // uniform: read after the barrier that follows every write
    // [WARPS][QT] maxima, sums, then [WARPS][8][CS] outputs, eight columns at a time
    float* xm = reinterpret_cast<float*>(smem);
    float* xl = xm + WARPS * QT;
    float* xo = xl + WARPS * QT;
    if (g == 0) {
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) {
        const int c = 8 * (i >> 1) + 2 * t + (i & 1);
        xm[warp * QT + c] = m[i];
        xl[warp * QT + c] = l[i];
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (n > 0) __syncthreads();
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        float* dst = xo + (warp * 8 + 2 * t) * CS + 16 * mt + g;
        dst[0] = o[mt][n][0];
        dst[CS] = o[mt][n][1];
        dst[8] = o[mt][n][2];
        dst[CS + 8] = o[mt][n][3];
      }
      __syncthreads();
      // 8 columns x 128 channels over 256 threads: four neighbouring channels a thread, a warp a column
      const int c = warp, d = 4 * lane;
      const int col = c0 + 8 * n + c;
      if (col <= clast) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, xm[w * QT + 8 * n + c]);
        float sum = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
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
        const int row = r0 + col / G, h = kvh * G + col % G;
        const int64_t at = (int64_t)row * args.HQ + h;
        if (args.splits == 1) {
          const float r = sum == 0.f ? 0.f : 1.f / sum;  // nothing visible: zeros
          *reinterpret_cast<uint2*>(args.out + at * D + d) = make_uint2(pack_bf16(y.x * r, y.y * r), pack_bf16(y.z * r, y.w * r));
        } else {
          const int64_t pt = (int64_t)split * sq_.T * args.HQ + at;
          *reinterpret_cast<float4*>(args.part_o + pt * D + d) = y;
          if (lane == 0) *reinterpret_cast<float2*>(args.part_ml + pt * 2) = make_float2(top, sum);
        }
      }
    }
    fence_proxy_async_smem();  // the exchange's writes come before the next tile's bulk copies
    __syncthreads();
  }
  if (tid == 0 && *abort_flag) atomicOr(&ffb_device_error_word, (uint32_t)ffb::ERR_ATTN_TIMEOUT);
}

// Joins the shares of one (row, head): one warp, four channels a lane.
// TC: the partials' columns are in the order that attention_kv4_tc.cu keeps them in.
template <bool TC>
__global__ void __launch_bounds__(256) kv4_combine_kernel(const AttnArgs args) {
  pdl_wait();
  pdl_launch();
  const int64_t n = (int64_t)args.seqs.T * args.HQ, at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= n) return;
  const int t = (int)(at / args.HQ), lane = threadIdx.x & 31;
  if (t < __ldg(args.seqs.row_start) || t >= __ldg(args.seqs.row_start + args.seqs.B)) return;
  float top = -INFINITY;
  for (int s = lane; s < args.splits; s += 32) top = fmaxf(top, args.part_ml[(s * n + at) * 2]);
  top = warp_max(top);
  float sum = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < args.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(args.part_ml + (s * n + at) * 2);
    const float* row = args.part_o + (s * n + at) * D;
    float4 v;
    if constexpr (TC) {
      // channel d = 64 half + 8 i + g sits in column 16 g + 8 half + 2 (i % 4) + i / 4
      const int half = lane >> 4, i = (lane >> 1) & 7, col = 64 * (lane & 1) + 8 * half + 2 * (i & 3) + (i >> 2);
      v = make_float4(row[col], row[col + 16], row[col + 32], row[col + 48]);
    } else {
      v = *reinterpret_cast<const float4*>(row + 4 * lane);
    }
    const float f = ml.x == -INFINITY && ml.y == 0.f ? 0.f : ex2(ml.x - top);
    sum = fmaf(ml.y, f, sum);
    y.x = fmaf(v.x, f, y.x);
    y.y = fmaf(v.y, f, y.y);
    y.z = fmaf(v.z, f, y.z);
    y.w = fmaf(v.w, f, y.w);
  }
  const float r = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(args.out + at * D + 4 * lane) = make_uint2(pack_bf16(y.x * r, y.y * r), pack_bf16(y.z * r, y.w * r));
}

// How a call is laid out.  kernel: 1 / 2 = the register path with 8 / 16 query columns a CTA,
// TC = the tensor-memory path with 256.
constexpr int TC = 3;
struct Plan {
  int kernel, tiles, splits;
};

// Shares of the page axis: enough CTAs for every SM, against the start and end of a CTA and the
// join.  slots: CTAs that run at once; step: pages a CTA takes at a time; step_us, cta_us: what
// such a step and a CTA's start and end take; join_us: a share's partials, written and read.
// Only share counts that fill whole waves are compared.
int plan_splits(int64_t base, int64_t pages, int slots, int step, double step_us, double cta_us, double join_us) {
  int best = 1;
  double best_cost = 0;
  for (int wave = 0; wave <= 4; ++wave) {
    int64_t fit = wave == 0 ? 1 : wave * slots / base;
    if (fit > pages / step) fit = pages / step;
    const int s = wave == 0 ? 1 : (int)(fit < 64 ? fit : 64);
    if (s < 1) continue;
    const double waves = (double)((base * s + slots - 1) / slots);
    const double rounds = (double)((pages + step * s - 1) / (step * s));
    const double cost = waves * (rounds * step_us + cta_us) + (s > 1 ? 2.0 + join_us * s : 0.0);
    if (wave == 0 || cost < best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}

Plan make_plan(int B, int T, int HQ, int HK, int max_rows, int max_pages, int window, int sinks) {
  Plan p;
  const int64_t cols = (int64_t)max_rows * (HQ / HK);
  p.kernel = cols <= 8 ? 1 : cols <= 16 ? 2 : TC;
  const int width = p.kernel == TC ? 256 : 8 * p.kernel;
  const int64_t tiles = (cols + width - 1) / width;
  p.tiles = (int)(tiles < 4096 ? tiles : 4096);
  int64_t pages = max_pages;
  if (window > 0) {
    const int64_t seen = ((int64_t)sinks + 63) / 64 + ((int64_t)window + max_rows + 126) / 64;
    if (seen < pages) pages = seen;
  }
  const double join = (double)T * HQ * (D + 2) * 4 * 2 / 5e6;  // written and read at about 5 TB/s
  const int64_t base = (int64_t)B * HK * p.tiles;
  const int sms = ffb::sm_count();
  p.splits = p.kernel == TC ? plan_splits(base, pages, sms, 2, 1.4, 5.0, join)
                            : plan_splits(base, pages, (p.kernel == 1 ? Shape<1>::PER_SM : Shape<2>::PER_SM) * sms, GROUPS, 0.9, 3.0, join);
  return p;
}

}  // namespace

namespace kv4 {
cudaError_t launch_attention_tc(const AttnArgs& a, unsigned grid_x, unsigned tiles, cudaStream_t stream);
}

extern "C" int64_t ffb_attention_kv4_workspace(int B, int T, int HQ, int HK, int max_rows, int max_pages, int window,
                                               int sinks) {
  if (B <= 0 || T <= 0 || HQ <= 0 || HK <= 0 || HQ % HK != 0 || max_rows <= 0 || max_pages <= 0 || window < 0 || sinks < 0)
    return 0;
  const Plan p = make_plan(B, T, HQ, HK, max_rows, max_pages, window, sinks);
  return p.splits > 1 ? (int64_t)p.splits * T * HQ * (D + 2) * 4 : 0;
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
  FFB_REQUIRE(isfinite(scale), "%s: scale must be finite", who);
  FFB_REQUIRE(window >= 0 && sinks >= 0 && window <= (1 << 30) && sinks <= (1 << 30), "%s: window %d, sinks %d", who,
              window, sinks);
  FFB_REQUIRE((int64_t)T * HQ <= (1 << 30), "%s: T=%d x HQ=%d too large", who, T, HQ);
  FFB_REQUIRE(sinks == 0 || window > 0, "%s: sinks without a window", who);
  FFB_REQUIRE(ffb::aligned(q, 16) && ffb::aligned(out, 16), "%s: q and out must be 16-byte aligned", who);
  const Plan p = make_plan(B, T, HQ, HK, max_rows, max_pages, window, sinks);
  const int64_t need = p.splits > 1 ? (int64_t)p.splits * T * HQ * (D + 2) * 4 : 0;
  FFB_REQUIRE(need == 0 || (ws && ws_bytes >= need && ffb::aligned(ws, 16)),
              "%s: workspace of %lld bytes (16-byte aligned) needed, %lld given", who, (long long)need, (long long)ws_bytes);
  const int64_t grid = (int64_t)B * HK * p.splits;
  FFB_REQUIRE(grid <= 0x7fffffff, "%s: B=%d HK=%d too large", who, B, HK);
  float* po = static_cast<float*>(ws);
  AttnArgs a = {q, out, po, po ? po + (int64_t)p.splits * T * HQ * D : nullptr,
            {const_cast<uint8_t*>(pages), page_table, row_start, ctx_len, num_pages, max_pages, B, T, HK, table_stride},
            HQ, p.splits, window, sinks, scale * 1.4426950408889634f};
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (p.kernel == TC) {
    e = kv4::launch_attention_tc(a, (unsigned)grid, p.tiles, st);
  } else {
    void (*kernel)(const AttnArgs) = p.kernel == 1 ? kv4_attention_kernel<1> : kv4_attention_kernel<2>;
    const int smem = p.kernel == 1 ? Shape<1>::SMEM : Shape<2>::SMEM;
    e = ffb::set_smem_attr(reinterpret_cast<const void*>(kernel), smem);
    if (e == cudaSuccess) e = ffb::launch(kernel, dim3((unsigned)grid, p.tiles), dim3(THREADS), smem, st, a);
  }
  if (e == cudaSuccess && p.splits > 1)
    e = ffb::launch(p.kernel == TC ? kv4_combine_kernel<true> : kv4_combine_kernel<false>,
                    dim3((unsigned)(((int64_t)T * HQ + 7) / 8)), dim3(256), 0, st, a);
  if (e != cudaSuccess) return ffb::fail(FFB_ECUDA, "%s: %s", who, cudaGetErrorString(e));
  return FFB_OK;
}
