// Writing and reading the 4-bit paged K/V cache (layout and quantiser: kv4.cuh).
//
// ffb_qk_norm_rope_kv4: the per-head RMSNorm and rotation of queries and keys
//   n = x / sqrt(mean(x^2) + eps) * w,  y[i] = n[i] c[i] - n[i + 64] s[i]   (i < 64)
//                                       y[i] = n[i] c[i] + n[i - 64] s[i]   (i >= 64)
// with the queries rounded once to bf16 and the keys and values quantised straight into the
// cache.  Sixteen lanes take one (row, head): lane i holds channels 4i..4i+3 and 64+4i..,
// so the rotation needs no exchange and a scale group is eight lanes.  Keys are computed in
// fp64 up to their codes: a key next to the border of two codes gets the same code whatever
// the order of operations (fp64 arithmetic is an eighth of the pass's heads' work).
// Bound by HBM: a row reads 256 (HQ + 2 HK) + 512 bytes and writes 256 HQ + 144 HK.
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
__device__ __forceinline__ double quotient(double x, double s) { return x / s; }
__device__ __forceinline__ float quotient(float x, float s) { return __fdiv_rn(x, s); }

// Scale and nibbles (lowest first) of this lane's four values of a group held by eight lanes.
template <typename F>
__device__ __forceinline__ uint32_t group_codes(const F (&y)[4], uint32_t mask, float& scale) {
  const F big = (F)1.7014118346046923e38;  // 2^127
  F top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const F a = y[e] < 0 ? -y[e] : y[e];
    top = a < big ? (a > top ? a : top) : (F)INFINITY;  // a NaN fails the comparison too
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const F other = __shfl_xor_sync(mask, top, o);
    top = other > top ? other : top;
  }
  if (!(top < big)) {
    scale = __uint_as_float(0x7fc00000u);
    return 0x8888u;
  }
  if (top < (F)7.888609052210118e-31) {  // 2^-100
    scale = 0.f;
    return 0x8888u;
  }
  const F s = up5(quotient(top, (F)7));
  scale = (float)s;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int q = (int)rint(quotient(y[e], s));
    codes |= (uint32_t)(min(max(q, -7), 7) + 8) << (4 * e);
  }
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

template <typename F>
__device__ __forceinline__ void norm_rotate(const float (&xa)[4], const float (&xb)[4], const uint16_t* w,
                                            const uint16_t* cr, const uint16_t* sr, float eps, int i, uint32_t mask,
                                            F (&ya)[4], F (&yb)[4]) {
  double ss = 0.0;  // bf16 squares are exact in fp32, their fp64 sum does not depend on its order
#pragma unroll
  for (int e = 0; e < 4; ++e) ss += (double)(xa[e] * xa[e]) + (double)(xb[e] * xb[e]);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
  const F inv = (F)(1.0 / sqrt(ss / D + (double)eps));
  float wa[4], wb[4], ca[4], cb[4], sa[4], sb[4];
  unpack4(__ldg(reinterpret_cast<const uint2*>(w + 4 * i)), wa);
  unpack4(__ldg(reinterpret_cast<const uint2*>(w + 64 + 4 * i)), wb);
  unpack4(__ldg(reinterpret_cast<const uint2*>(cr + 4 * i)), ca);
  unpack4(__ldg(reinterpret_cast<const uint2*>(cr + 64 + 4 * i)), cb);
  unpack4(__ldg(reinterpret_cast<const uint2*>(sr + 4 * i)), sa);
  unpack4(__ldg(reinterpret_cast<const uint2*>(sr + 64 + 4 * i)), sb);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const F na = (F)xa[e] * inv * (F)wa[e], nb = (F)xb[e] * inv * (F)wb[e];
    ya[e] = na * (F)ca[e] - nb * (F)sa[e];
    yb[e] = nb * (F)cb[e] + na * (F)sb[e];
  }
}

__global__ void __launch_bounds__(WARPS * 32) kv4_write_kernel(const WriteArgs p) {
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, i = lane & 15;
  const uint32_t mask = 0xffffu << (lane & 16);
  const int heads = p.HQ + 2 * p.seqs.HK;
  const int64_t item = ((int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5)) * 2 + (lane >> 4);
  if (item >= (int64_t)p.seqs.T * heads) return;
  const int t = (int)(item / heads), h = (int)(item - (int64_t)t * heads);
  const int b = seq_of(p.seqs, t);
  if (b < 0) return;
  float xa[4], xb[4];
  const uint16_t* x = p.qkv + t * p.row_stride + (int64_t)h * D;
  unpack4(*reinterpret_cast<const uint2*>(x + 4 * i), xa);
  unpack4(*reinterpret_cast<const uint2*>(x + 64 + 4 * i), xb);
  const uint16_t* cr = p.cos + (int64_t)t * D;
  const uint16_t* sr = p.sin + (int64_t)t * D;
  if (h < p.HQ) {
    float ya[4], yb[4];
    norm_rotate(xa, xb, p.q_norm, cr, sr, p.eps, i, mask, ya, yb);
    uint16_t* dst = p.yq + ((int64_t)h * p.seqs.T + t) * D;
    *reinterpret_cast<uint2*>(dst + 4 * i) =
        make_uint2((uint32_t)f2bf(ya[0]) | ((uint32_t)f2bf(ya[1]) << 16), (uint32_t)f2bf(ya[2]) | ((uint32_t)f2bf(ya[3]) << 16));
    *reinterpret_cast<uint2*>(dst + 64 + 4 * i) =
        make_uint2((uint32_t)f2bf(yb[0]) | ((uint32_t)f2bf(yb[1]) << 16), (uint32_t)f2bf(yb[2]) | ((uint32_t)f2bf(yb[3]) << 16));
    return;
  }
  const bool is_v = h >= p.HQ + p.seqs.HK;
  const int kvh = h - p.HQ - (is_v ? p.seqs.HK : 0);
  const int64_t pos = (int64_t)__ldg(p.seqs.ctx_len + b) - (__ldg(p.seqs.row_start + b + 1) - t);
  uint8_t* rec = record_of(p.seqs, b, pos, kvh);
  if (!rec) {
    if (i == 0) atomicOr(&ffb_device_error_word, (uint32_t)ffb::ERR_KV4_PAGE);
    return;
  }
  const int token = (int)(pos % PAGE);
  float s_lo, s_hi;
  uint32_t lo, hi;
  if (is_v) {
    lo = group_codes(xa, mask, s_lo);
    hi = group_codes(xb, mask, s_hi);
    store_v(rec + V_CODES + 64 * token, lo, hi, i, token, mask);
  } else {
    double ya[4], yb[4];
    norm_rotate(xa, xb, p.k_norm, cr, sr, p.eps, i, mask, ya, yb);
    lo = group_codes(ya, mask, s_lo);
    hi = group_codes(yb, mask, s_hi);
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
  const int64_t item = ((int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5)) * 2 + (lane >> 4);
  if (item >= (int64_t)p.T * p.HK) return;
  const int h = (int)(item / p.T), t = (int)(item - (int64_t)h * p.T);
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
  WriteArgs a = {qkv, row_stride, q_norm, k_norm, cos, sin, yq, eps, HQ,
                 {pages, page_table, row_start, ctx_len, num_pages, max_pages, B, T, HK, table_stride}};
  const int64_t items = (int64_t)T * (HQ + 2 * HK), grid = (items + 2 * WARPS - 1) / (2 * WARPS);
  FFB_REQUIRE(grid <= 0x7fffffff, "%s: T=%d HQ=%d HK=%d too large", who, T, HQ, HK);
  cudaError_t e = ffb::launch(kv4_write_kernel, dim3((unsigned)grid), dim3(WARPS * 32), 0, (cudaStream_t)stream, a);
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
  const int64_t items = (int64_t)T * HK, grid = (items + 2 * WARPS - 1) / (2 * WARPS);
  FFB_REQUIRE(grid <= 0x7fffffff, "%s: T=%d HK=%d too large", who, T, HK);
  cudaError_t e = ffb::launch(kv4_read_kernel, dim3((unsigned)grid), dim3(WARPS * 32), 0, (cudaStream_t)stream, a, k, v);
  if (e != cudaSuccess) return ffb::fail(FFB_ECUDA, "%s: %s", who, cudaGetErrorString(e));
  return FFB_OK;
}
