// Writing and reading the 4-bit paged K/V cache (layout and quantiser: kv4.cuh).
//
// ffb_qk_norm_rope_kv4: the per-head RMSNorm and rotation of queries and keys
//   n = x / sqrt(mean(x^2) + eps) * w,  y[i] = n[i] c[i] - n[i + 64] s[i]   (i < 64)
//                                       y[i] = n[i] c[i] + n[i - 64] s[i]   (i >= 64)
// with the queries rounded once to bf16 and the keys and values quantised straight into the
// cache.  A row reads 256 (HQ + 2 HK) + 512 bytes and writes 256 HQ + 144 HK.
// Sixteen lanes take one (row, head): lane i holds channels 4i..4i+3 and 64+4i.., so the
// rotation needs no exchange and a scale group is eight lanes.  A CTA takes one row: the first
// ones of a row its query heads (four to a half warp once there are enough rows, their loads
// issued together), the last its key and value heads; a row's CTAs are launched next to each
// other, so that the quantiser's arithmetic runs beside the queries' traffic (behind it: 78 us
// where this takes 74.6).
// Measured: 7128 rows of 64 + 8 heads (275 MB) 69.9 us, 3.9 TB/s (in four sequences 71.5), of which the
// queries alone would take 45; 79% of the issue slots are used: the rest is the codes' instructions.  One row
// of 32 + 8 heads 2.8 us, 320 rows 5.9 us: launch and latency.  Reading those 7128 rows back 10.6 us, 3.5
// TB/s: a lane has one word of K and one of V on their way.
//
// The codes are those of the formula in exact arithmetic, up to fp64's rounding: a key next to
// the border of two codes must not fall to either side by chance.  Keys are worked out in fp32 with
// a bound on the error, and again in fp64 where a value lies within it of a border (about one head in
// 200).  Values are bf16: x - q s is exact, so borders are seen as such.
#include "kv4.cuh"
#include "pdl.cuh"

namespace {

using namespace kv4;
constexpr int WARPS = 8;

__device__ __forceinline__ void unpack4(uint2 u, float (&x)[4]) {
  x[0] = __uint_as_float(u.x << 16);
  x[1] = __uint_as_float(u.x & 0xffff0000u);
  x[2] = __uint_as_float(u.y << 16);
  x[3] = __uint_as_float(u.y & 0xffff0000u);
}

// Rounds a positive finite value up to five significant bits.
__device__ __forceinline__ double up5(double v) {
  const long long b = __double_as_longlong(v), low = (1ll << 48) - 1;
  return __longlong_as_double((b + low) & ~low);
}
__device__ __forceinline__ float up5(float v) {
  const uint32_t b = __float_as_uint(v), low = (1u << 19) - 1;
  return __uint_as_float((b + low) & ~low);
}
__device__ __forceinline__ float group_max(float top, uint32_t mask) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, o));
  return top;
}
constexpr float BIG = 1.7014118346046923e38f;    // 2^127
constexpr float SMALL = 7.888609052210118e-31f;  // 2^-100

// Scale and nibbles (lowest first) of this lane's four values of a group held by eight lanes.
// Values: bf16, exact.
__device__ __forceinline__ uint32_t value_codes(const float (&y)[4], uint32_t mask, float& scale) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = fabsf(y[e]) < BIG ? fmaxf(top, fabsf(y[e])) : INFINITY;  // a NaN fails it too
  top = group_max(top, mask);
  if (!(top < BIG) || top < SMALL) {
    scale = top < BIG ? 0.f : __uint_as_float(0x7fc00000u);
    return 0x8888u;
  }
  // (a bf16 over 7 is never so near a number of five bits that fp32's quotient crosses it)
  const float s = up5(__fdiv_rn(top, 7.f)), r = __frcp_rn(s), half = 0.5f * s;
  scale = s;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // q from the approximate quotient is one off at most; the rest x - q s is exact and tells
    float q = rintf(y[e] * r);
    const float rest = fmaf(-q, s, y[e]), off = fabsf(rest);
    if (off > half || (off == half && ((int)q & 1))) q += rest > 0.f ? 1.f : -1.f;
    codes |= (uint32_t)((int)fminf(fmaxf(q, -7.f), 7.f) + 8) << (4 * e);
  }
  return codes;
}
// Keys, in fp32: y is within 9.5 x 2^-24 of the formula's value, so a quotient y / s <= 7 within
// 11.5 x 2^-24 x 7 < 1e-5 and max / 7 within 10.5 units of its last place.  `doubt`: fp32 cannot tell on
// which side of a border a value lies, or the group's range is not its own.
__device__ __forceinline__ uint32_t key_codes(const float (&d)[4], float inv, uint32_t mask, float& scale, bool& doubt) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = fabsf(d[e]) < 1e36f ? fmaxf(top, fabsf(d[e])) : INFINITY;
  top = group_max(top, mask);
  const float most = top * inv, seventh = __fdiv_rn(most, 7.f), s = up5(seventh);
  doubt |= !(top > 1e-30f && top < 1e36f && most > 1e-29f && most < 1e37f) ||
           ((__float_as_uint(seventh) + 16u) & ((1u << 19) - 1)) < 32u;
  const float r = __frcp_rn(s);
  scale = s;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float t = d[e] * inv * r, q = rintf(t);
    doubt |= fabsf(fabsf(t - q) - 0.5f) < 1e-5f;
    codes |= (uint32_t)((int)fminf(fmaxf(q, -7.f), 7.f) + 8) << (4 * e);
  }
  return codes;
}
// Keys, in fp64: the formula as it stands.
__device__ __forceinline__ uint32_t key_codes(const double (&y)[4], uint32_t mask, float& scale) {
  double top = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = fabs(y[e]) < (double)BIG ? fmax(top, fabs(y[e])) : (double)INFINITY;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = fmax(top, __shfl_xor_sync(mask, top, o));
  if (!(top < (double)BIG) || top < (double)SMALL) {
    scale = top < (double)BIG ? 0.f : __uint_as_float(0x7fc00000u);
    return 0x8888u;
  }
  const double s = up5(top / 7.0);
  scale = (float)s;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) codes |= (uint32_t)((int)fmin(fmax(rint(y[e] / s), -7.0), 7.0) + 8) << (4 * e);
  return codes;
}

// The 64 code bytes of one token: lane i gives nibbles of channels 4i.. (lo) and 64+4i.. (hi)
// and stores one 4-byte word.
__device__ __forceinline__ void store_k(uint8_t* dst, uint32_t lo, uint32_t hi, int i, uint32_t mask) {
  const bool odd = i & 1;
  const uint32_t got = __shfl_xor_sync(mask, odd ? lo : hi, 1);
  const uint32_t word = odd ? (got | (hi << 16)) : (lo | (got << 16));
  // word 4 t + j: t = (i % 8) / 2, j = i / 8 (low channels) or 2 + i / 8
  *reinterpret_cast<uint32_t*>(dst + 16 * ((i & 7) >> 1) + 4 * ((i >> 3) + (odd ? 2 : 0))) = word;
}
__device__ __forceinline__ void store_v(uint8_t* dst, uint32_t lo, uint32_t hi, int i, int token, uint32_t mask) {
  // chunk g = 4 (i % 2) + e, its nibble i / 2 (word 0, low channels) or 8 + i / 2 (word 1):
  // the eight lanes of one parity reduce 8 words so that each ends with one of them
  uint32_t w[8];
  const int sh = 4 * (i >> 1);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[2 * e] = ((lo >> (4 * e)) & 15u) << sh;
    w[2 * e + 1] = ((hi >> (4 * e)) & 15u) << sh;
  }
  const int id = i >> 1;
#pragma unroll
  for (int step = 0; step < 3; ++step) {
    const int n = 4 >> step;
    const bool up = (id >> step) & 1;
#pragma unroll
    for (int k = 0; k < n; ++k) {
      const uint32_t got = __shfl_xor_sync(mask, up ? w[k] : w[k + n], 2 << step);
      w[k] = (up ? w[k + n] : w[k]) | got;
    }
  }
  const int which = ((id & 1) << 2) | (id & 2) | (id >> 2);  // 2 e + word
  const int g = 4 * (i & 1) + (which >> 1);
  *reinterpret_cast<uint32_t*>(dst + 8 * (g ^ (token & 4)) + 4 * (which & 1)) = w[0];
}

struct WriteArgs {
  const uint16_t* qkv;
  int64_t row_stride;
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  const uint16_t* cos;
  const uint16_t* sin;
  uint16_t* yq;
  float eps;
  int HQ;
  Seqs seqs;
};

// Sum over the sixteen lanes of one (row, head).
template <typename F>
__device__ __forceinline__ F head_sum(F v, uint32_t mask) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) v += __shfl_xor_sync(mask, v, o);
  return v;
}

struct Turn {  // this lane's cosines and sines of a row
  float ca[4], cb[4], sa[4], sb[4];
};
__device__ __forceinline__ void load_turn(const WriteArgs& p, int t, int i, Turn& r) {
  const int64_t at = (int64_t)t * D + 4 * i;
  unpack4(__ldg(reinterpret_cast<const uint2*>(p.cos + at)), r.ca);
  unpack4(__ldg(reinterpret_cast<const uint2*>(p.cos + at + 64)), r.cb);
  unpack4(__ldg(reinterpret_cast<const uint2*>(p.sin + at)), r.sa);
  unpack4(__ldg(reinterpret_cast<const uint2*>(p.sin + at + 64)), r.sb);
}

// A head's values after norm and rotation in fp64, from the inputs: lane i's channels 4i.. and 64+4i...
__device__ __forceinline__ void exact_head(const uint2* x, const uint2* w, const uint2* c, const uint2* s, float eps, int i,
                                           uint32_t mask, double (&ya)[4], double (&yb)[4]) {
  float xa[4], xb[4], wa[4], wb[4], ca[4], cb[4], sa[4], sb[4];
  unpack4(__ldg(x + i), xa);
  unpack4(__ldg(x + 16 + i), xb);
  unpack4(__ldg(w + i), wa);
  unpack4(__ldg(w + 16 + i), wb);
  unpack4(__ldg(c + i), ca);
  unpack4(__ldg(c + 16 + i), cb);
  unpack4(__ldg(s + i), sa);
  unpack4(__ldg(s + 16 + i), sb);
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) sum += (double)xa[e] * (double)xa[e] + (double)xb[e] * (double)xb[e];
  const double norm = 1.0 / sqrt(head_sum(sum, mask) / D + (double)eps);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double na = (double)xa[e] * norm * (double)wa[e], nb = (double)xb[e] * norm * (double)wb[e];
    ya[e] = na * (double)ca[e] - nb * (double)sa[e];
    yb[e] = nb * (double)cb[e] + na * (double)sb[e];
  }
}
__device__ __forceinline__ void store_query(uint16_t* dst, const float (&ya)[4], const float (&yb)[4]) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(ya[0], ya[1]), pack_bf16(ya[2], ya[3]));
  *reinterpret_cast<uint2*>(dst + 64) = make_uint2(pack_bf16(yb[0], yb[1]), pack_bf16(yb[2], yb[3]));
}
// Whether fp32 holds a query's mean square plus eps, and the squares that count in it.
constexpr float MOST = 1e33f;
__device__ __forceinline__ bool in_range(float mean) { return mean > SMALL && mean < MOST; }
__device__ __forceinline__ const uint2* query_of(const WriteArgs& p, int t, int h) {
  return reinterpret_cast<const uint2*>(p.qkv + (int64_t)t * p.row_stride + (int64_t)h * D);
}
// A query that is not in range (values of 2^55 and more, or tiny ones with an eps as small): in fp64.
__device__ __forceinline__ void far_query(const WriteArgs& p, int t, int h, int i, uint32_t mask) {
  double da[4], db[4];
  float ya[4], yb[4];
  exact_head(query_of(p, t, h), reinterpret_cast<const uint2*>(p.q_norm), reinterpret_cast<const uint2*>(p.cos + (int64_t)t * D),
             reinterpret_cast<const uint2*>(p.sin + (int64_t)t * D), p.eps, i, mask, da, db);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    ya[e] = (float)da[e];
    yb[e] = (float)db[e];
  }
  store_query(p.yq + ((int64_t)h * p.seqs.T + t) * D + 4 * i, ya, yb);
}
// Those of this half warp's U heads, found again from the inputs: the caller keeps no register for it.
template <int U>
__device__ __noinline__ void far_queries(const WriteArgs& p) {
  const int i = threadIdx.x & 15, t = (int)(blockIdx.z * gridDim.y + blockIdx.y);
  const int h0 = (int)(blockIdx.x * 2 * WARPS + (threadIdx.x >> 4)) * U;
  const uint32_t mask = 0xffffu << (threadIdx.x & 16);
#pragma unroll 1
  for (int h = h0; h < min(h0 + U, p.HQ); ++h) {
    const uint2* x = query_of(p, t, h);
    float xa[4], xb[4], ss = 0.f;
    unpack4(__ldg(x + i), xa);
    unpack4(__ldg(x + 16 + i), xb);
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = fmaf(xa[e], xa[e], fmaf(xb[e], xb[e], ss));
    if (!in_range(head_sum(ss, mask) * (1.f / D) + p.eps)) far_query(p, t, h, i, mask);
  }
}

// The codes of one key, lane i's low and high ones, and the scales of its two groups.
struct KeyCodes {
  uint32_t lo, hi;
  float s_lo, s_hi;
};
__device__ __forceinline__ KeyCodes exact_key(const uint2* x, const uint2* w, const uint2* c, const uint2* s, float eps, int i,
                                           uint32_t mask) {
  double ya[4], yb[4];
  exact_head(x, w, c, s, eps, i, mask, ya, yb);
  KeyCodes k;
  k.lo = key_codes(ya, mask, k.s_lo);
  k.hi = key_codes(yb, mask, k.s_hi);
  return k;
}

// Called, it takes no registers of the common path: a fifth CTA an SM for long calls (7128 rows of 64 + 8
// heads: 4 us of 70).  Where every CTA is resident anyway it is inline (320 rows: 0.5 us of 6).
__device__ __noinline__ KeyCodes exact_key_call(const uint2* x, const uint2* w, const uint2* c, const uint2* s, float eps,
                                                int i, uint32_t mask) {
  return exact_key(x, w, c, s, eps, i, mask);
}

// U: query heads of a half warp.
template <int U>
__global__ void __launch_bounds__(WARPS * 32, U > 1 ? 5 : 4) kv4_write_kernel(const __grid_constant__ WriteArgs p, int q_chunks) {
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, i = lane & 15, slot = threadIdx.x >> 4;
  const int t = (int)(blockIdx.z * gridDim.y + blockIdx.y), chunk = (int)blockIdx.x;  // a row's CTAs next to each other
  if (t >= p.seqs.T) return;
  const uint32_t mask = 0xffffu << (lane & 16);
  const int HK = p.seqs.HK;
  const uint16_t* x = p.qkv + (int64_t)t * p.row_stride + 4 * i;
  if (chunk < q_chunks) {
    const int h0 = (chunk * 2 * WARPS + slot) * U;
    uint2 ua[U], ub[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ua[u] = ub[u] = make_uint2(0u, 0u);
      if (h0 + u < p.HQ) {
        ua[u] = __ldg(reinterpret_cast<const uint2*>(x + (int64_t)(h0 + u) * D));
        ub[u] = __ldg(reinterpret_cast<const uint2*>(x + (int64_t)(h0 + u) * D + 64));
      }
    }
    Turn r;
    load_turn(p, t, i, r);
    float wa[4], wb[4];
    unpack4(__ldg(reinterpret_cast<const uint2*>(p.q_norm + 4 * i)), wa);
    unpack4(__ldg(reinterpret_cast<const uint2*>(p.q_norm + 64 + 4 * i)), wb);
    if (t < __ldg(p.seqs.row_start) || t >= __ldg(p.seqs.row_start + p.seqs.B)) return;
    auto query = [&](int u) { return p.yq + ((int64_t)(h0 + u) * p.seqs.T + t) * D + 4 * i; };
    float means = 0.f;  // looked at once for all heads: a branch a head keeps their arithmetic apart
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h0 + u >= p.HQ) break;
      float xa[4], xb[4], ss = 0.f;
      unpack4(ua[u], xa);
      unpack4(ub[u], xb);
#pragma unroll
      for (int e = 0; e < 4; ++e) ss = fmaf(xa[e], xa[e], fmaf(xb[e], xb[e], ss));
      const float mean = head_sum(ss, mask) * (1.f / D) + p.eps;
      const float inv = __frsqrt_rn(mean);
      if (U > 1) {
        means += mean;
      } else if (!in_range(mean)) {  // before the store: a call of one row may write over its inputs
        far_query(p, t, h0, i, mask);
        break;
      }
      float ya[4], yb[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float na = xa[e] * inv * wa[e], nb = xb[e] * inv * wb[e];
        ya[e] = na * r.ca[e] - nb * r.sa[e];
        yb[e] = nb * r.cb[e] + na * r.sb[e];
      }
      store_query(query(u), ya, yb);
    }
    if (U > 1 && !(means < MOST && p.eps > SMALL)) far_queries<U>(p);
    return;
  }
  const int pair = (chunk - q_chunks) * 2 * WARPS + slot;
  if (pair >= 2 * HK) return;
  const bool is_v = pair >= HK;
  const int h = is_v ? pair - HK : pair;
  const uint2 ua = __ldg(reinterpret_cast<const uint2*>(x + (int64_t)(p.HQ + pair) * D));
  const uint2 ub = __ldg(reinterpret_cast<const uint2*>(x + (int64_t)(p.HQ + pair) * D + 64));
  const int b = seq_of(p.seqs, t);
  if (b < 0) return;
  const int64_t pos = (int64_t)__ldg(p.seqs.ctx_len + b) - (__ldg(p.seqs.row_start + b + 1) - t);
  uint8_t* rec = record_of(p.seqs, b, pos, h);
  if (!rec) {
    if (i == 0) atomicOr(&ffb_device_error_word, (uint32_t)ffb::ERR_KV4_PAGE);
    return;
  }
  const int token = (int)(pos & (PAGE - 1));
  float xa[4], xb[4], s_lo, s_hi;
  unpack4(ua, xa);
  unpack4(ub, xb);
  if (is_v) {
    const uint32_t lo = value_codes(xa, mask, s_lo), hi = value_codes(xb, mask, s_hi);
    store_v(rec + V_CODES + 64 * token, lo, hi, i, token, mask);
  } else {
    Turn r;
    load_turn(p, t, i, r);
    float wa[4], wb[4], ss = 0.f, da[4], db[4];
    unpack4(__ldg(reinterpret_cast<const uint2*>(p.k_norm + 4 * i)), wa);
    unpack4(__ldg(reinterpret_cast<const uint2*>(p.k_norm + 64 + 4 * i)), wb);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ss = fmaf(xa[e], xa[e], fmaf(xb[e], xb[e], ss));
      // x w has 16 bits and x w c 24: only the sum rounds
      const float ta = xa[e] * wa[e], tb = xb[e] * wb[e];
      da[e] = fmaf(ta, r.ca[e], -(tb * r.sa[e]));
      db[e] = fmaf(tb, r.cb[e], ta * r.sb[e]);
    }
    ss = head_sum(ss, mask);
    const float inv = __frsqrt_rn(ss * (1.f / D) + p.eps);
    bool doubt = !(ss > 1e-20f && ss < 1e30f);
    uint32_t lo = key_codes(da, inv, mask, s_lo, doubt), hi = key_codes(db, inv, mask, s_hi, doubt);
    if (__any_sync(mask, doubt)) {  // about one head in 200
      const uint2* kx = reinterpret_cast<const uint2*>(p.qkv + (int64_t)t * p.row_stride + (int64_t)(p.HQ + pair) * D);
      const uint2* kw = reinterpret_cast<const uint2*>(p.k_norm);
      const uint2* kc = reinterpret_cast<const uint2*>(p.cos + (int64_t)t * D);
      const uint2* ks = reinterpret_cast<const uint2*>(p.sin + (int64_t)t * D);
      const KeyCodes k = U > 1 ? exact_key_call(kx, kw, kc, ks, p.eps, i, mask) : exact_key(kx, kw, kc, ks, p.eps, i, mask);
      lo = k.lo;
      hi = k.hi;
      s_lo = k.s_lo;
      s_hi = k.s_hi;
    }
    store_k(rec + 64 * token, lo, hi, i, mask);
  }
  if ((i & 7) == 0) {  // groups i / 8 (low channels) and 2 + i / 8
    uint16_t* sc = reinterpret_cast<uint16_t*>(rec + (is_v ? V_SCALES : K_SCALES)) + 4 * token + (i >> 3);
    sc[0] = f2bf(s_lo);
    sc[2] = f2bf(s_hi);
  }
}

// Sixteen lanes per (row, head): lane i reads one word of K and of V and stores 8 channels of
// each (16 bytes).
__global__ void __launch_bounds__(WARPS * 32) kv4_read_kernel(const Seqs p, uint16_t* k, uint16_t* v) {
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, i = lane & 15;
  const uint32_t mask = 0xffffu << (lane & 16);
  const int t = (int)blockIdx.x * 2 * WARPS + (threadIdx.x >> 4), h = blockIdx.y;
  if (t >= p.T) return;
  const int b = seq_of(p, t);
  if (b < 0) return;
  const int64_t pos = (int64_t)__ldg(p.ctx_len + b) - (__ldg(p.row_start + b + 1) - t);
  const uint8_t* rec = record_of(p, b, pos, h);
  uint16_t* dk = k + ((int64_t)h * p.T + t) * D;
  uint16_t* dv = v + ((int64_t)h * p.T + t) * D;
  if (!rec) {
    if (i == 0) atomicOr(&ffb_device_error_word, (uint32_t)ffb::ERR_KV4_PAGE);
    *reinterpret_cast<uint4*>(dk + 8 * i) = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(dv + 8 * i) = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const int token = (int)(pos % PAGE);
  const uint32_t wk = *reinterpret_cast<const uint32_t*>(rec + 64 * token + 4 * i);
  const uint32_t wv = *reinterpret_cast<const uint32_t*>(rec + V_CODES + 64 * token + 4 * i);
  const uint16_t* ks = reinterpret_cast<const uint16_t*>(rec + K_SCALES) + 4 * token;
  const uint16_t* vs = reinterpret_cast<const uint16_t*>(rec + V_SCALES) + 4 * token;
  const float sk = bf2f(ks[i & 3]), sv = bf2f(vs[i >> 2]);
  uint32_t ok[4], ov[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {  // exact products: the casts round nothing
    const float a = (float)((int)((wk >> (8 * e)) & 15u) - 8) * sk, c = (float)((int)((wk >> (8 * e + 4)) & 15u) - 8) * sk;
    ok[e] = (uint32_t)f2bf(a) | ((uint32_t)f2bf(c) << 16);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // channel 8 i + g: nibble i of chunk g
    float y[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int g = 2 * e + u;
      const uint32_t w = __shfl_sync(mask, wv, 2 * (g ^ (token & 4)) + (i >> 3), 16);
      y[u] = (float)((int)((w >> (4 * (i & 7))) & 15u) - 8) * sv;
    }
    ov[e] = (uint32_t)f2bf(y[0]) | ((uint32_t)f2bf(y[1]) << 16);
  }
  *reinterpret_cast<uint4*>(dk + 32 * (i & 3) + 8 * (i >> 2)) = make_uint4(ok[0], ok[1], ok[2], ok[3]);
  *reinterpret_cast<uint4*>(dv + 8 * i) = make_uint4(ov[0], ov[1], ov[2], ov[3]);
}

}  // namespace

namespace ffb {
int kv4_check(const char* who, const void* pages, const int* table, const int* row_start, const int* ctx_len,
              int num_pages, int64_t table_stride, int max_pages, int B, int T, int HK) {
  FFB_REQUIRE(pages && table && row_start && ctx_len, "%s: NULL pointer", who);
  FFB_REQUIRE(num_pages > 0 && max_pages > 0 && B > 0 && T > 0 && HK > 0,
              "%s: bad shape pages=%d table width=%d B=%d T=%d HK=%d", who, num_pages, max_pages, B, T, HK);
  FFB_REQUIRE(max_pages <= FFB_KV4_MAX_PAGES, "%s: table width %d (at most %d)", who, max_pages, FFB_KV4_MAX_PAGES);
  FFB_REQUIRE(B <= 65535 && T <= (1 << 24) && HK <= 1024, "%s: B=%d T=%d HK=%d too large", who, B, T, HK);
  FFB_REQUIRE(table_stride >= max_pages || B == 1, "%s: table stride %lld < width %d", who, (long long)table_stride,
              max_pages);
  FFB_REQUIRE(aligned(pages, 16), "%s: pages must be 16-byte aligned", who);
  FFB_REQUIRE(aligned(table, 4) && aligned(row_start, 4) && aligned(ctx_len, 4), "%s: index alignment", who);
  return FFB_OK;
}
}  // namespace ffb

extern "C" int ffb_qk_norm_rope_kv4(const uint16_t* qkv, int64_t row_stride, const uint16_t* q_norm,
                                    const uint16_t* k_norm, float eps, const uint16_t* cos, const uint16_t* sin,
                                    uint16_t* yq, uint8_t* pages, int num_pages, const int* page_table,
                                    int64_t table_stride, int max_pages, const int* row_start, const int* ctx_len,
                                    int B, int T, int HQ, int HK, void* stream) {
  const char* who = "ffb_qk_norm_rope_kv4";
  int rc = ffb::kv4_check(who, pages, page_table, row_start, ctx_len, num_pages, table_stride, max_pages, B, T, HK);
  if (rc) return rc;
  FFB_REQUIRE(qkv && q_norm && k_norm && cos && sin && yq, "%s: NULL pointer", who);
  FFB_REQUIRE(HQ > 0 && HQ % HK == 0 && HQ <= 4096, "%s: bad heads HQ=%d HK=%d", who, HQ, HK);
  FFB_REQUIRE(row_stride >= (int64_t)(HQ + 2 * HK) * D && row_stride % 4 == 0, "%s: row_stride %lld", who,
              (long long)row_stride);
  FFB_REQUIRE(eps >= 0.f, "%s: eps %g", who, (double)eps);
  FFB_REQUIRE(ffb::aligned(qkv, 8) && ffb::aligned(q_norm, 8) && ffb::aligned(k_norm, 8) && ffb::aligned(cos, 8) &&
                  ffb::aligned(sin, 8) && ffb::aligned(yq, 8),
              "%s: qkv, norms, tables and yq must be 8-byte aligned", who);
  FFB_REQUIRE((T == 1 && yq == qkv) || !ffb::overlap(yq, (int64_t)T * HQ * D * 2, qkv,
                                                      ((T - 1) * row_stride + (int64_t)(HQ + 2 * HK) * D) * 2),
              "%s: yq and qkv overlap", who);
  WriteArgs a = {qkv, row_stride, q_norm, k_norm, cos, sin, yq, eps, HQ,
                 {pages, page_table, row_start, ctx_len, num_pages, max_pages, B, T, HK, table_stride}};
  // us with one / four query heads a half warp, 64 + 8 heads: 148 rows 4.8 / 5.0, 320 7.2 / 6.3, 592 10.3 / 8.7,
  // 7128 111 / 70; 16 + 8 heads: 320 rows 5.0 / 5.5, 592 7.1 / 7.4, 2400 19.1 / 19.0, 7128 56 / 50.  The rule
  // is one for all heads: four from four rows an SM on
  const bool many = T >= 4 * ffb::sm_count();
  const int heads = (many ? 4 : 1) * 2 * WARPS, q_chunks = (HQ + heads - 1) / heads;
  const int rows = T < 65535 ? T : 65535;
  const dim3 grid(q_chunks + (2 * HK + 2 * WARPS - 1) / (2 * WARPS), rows, (T + rows - 1) / rows);
  cudaError_t e = many ? ffb::launch(kv4_write_kernel<4>, grid, dim3(WARPS * 32), 0, (cudaStream_t)stream, a, q_chunks)
                       : ffb::launch(kv4_write_kernel<1>, grid, dim3(WARPS * 32), 0, (cudaStream_t)stream, a, q_chunks);
  if (e != cudaSuccess) return ffb::fail(FFB_ECUDA, "%s: %s", who, cudaGetErrorString(e));
  return FFB_OK;
}

extern "C" int ffb_kv4_read(const uint8_t* pages, int num_pages, const int* page_table, int64_t table_stride,
                            int max_pages, const int* row_start, const int* ctx_len, uint16_t* k, uint16_t* v, int B,
                            int T, int HK, void* stream) {
  const char* who = "ffb_kv4_read";
  int rc = ffb::kv4_check(who, pages, page_table, row_start, ctx_len, num_pages, table_stride, max_pages, B, T, HK);
  if (rc) return rc;
  FFB_REQUIRE(k && v, "%s: NULL pointer", who);
  FFB_REQUIRE(ffb::aligned(k, 16) && ffb::aligned(v, 16), "%s: k and v must be 16-byte aligned", who);
  Seqs a = {const_cast<uint8_t*>(pages), page_table, row_start, ctx_len, num_pages, max_pages, B, T, HK, table_stride};
  const dim3 grid((T + 2 * WARPS - 1) / (2 * WARPS), HK);
  cudaError_t e = ffb::launch(kv4_read_kernel, grid, dim3(WARPS * 32), 0, (cudaStream_t)stream, a, k, v);
  if (e != cudaSuccess) return ffb::fail(FFB_ECUDA, "%s: %s", who, cudaGetErrorString(e));
  return FFB_OK;
}
