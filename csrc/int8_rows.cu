// Row quantisers of the 8-bit integer (W8A8) path: one scale per token, symmetric codes.
//
//   s = max(max_k |y_k| / 127, 2^-120),   q_k = rint(y_k / s)   (half to even, |q| <= 127)
//
// For rows that are read (vg_quant_int8) q is that of the exact quotient 127 y / max|y|, so that no rounding decides a code.
// For rows that are computed here y has rounding errors of its own, and q is rint(y * (1 / s)), which may differ from
// rint(y / s) where y / s is within 2^-16 of a half.
//
//   vg_quant_int8         y = x                                       (bf16 / f16 / f32 rows)
//   vg_add_rmsnorm_int8   res += delta;  y = res * rsqrt(mean res^2 + eps) * (w [+ 1])
//   vg_swiglu_int8        y = silu(gate) * up
//   vg_dequant_int8       q * s back to bf16 / f16 / f32
//
// The row is read once and stays in registers as fp32 between the reduction and the stores, so each kernel moves its
// inputs and outputs once and nothing else. A row that holds an infinity or a NaN (or whose sum of squares leaves
// fp32) gets scale NaN and codes 0: everything computed from it is NaN instead of a plausible wrong number. The floor
// of the scale keeps an all-zero row at codes 0 and 1 / s finite.
// Inputs are read with ordinary loads: a kernel may start before its predecessor has written them, so they are not
// read-only for its lifetime, which ld.global.nc (restrict pointers, __ldg) asks for.
#include <atomic>

#include "common.cuh"
#include "api.h"

namespace {
using namespace vg;

constexpr int MAX_CLUSTER = 8;
constexpr int RING_SLOTS = 8;
constexpr int RING_GROUPS = 2560;                         // groups of eight of the widest row of the ring form
// Largest row width: a cluster of eight CTAs of 1024 threads with two (three) groups of eight each.
constexpr int ROW_MAX = MAX_CLUSTER * 1024 * 2 * 8;
constexpr float INT8_MAX_CODE = 127.0f;
constexpr float AMAX_FLOOR = 127.0f * 0x1p-120f;          // exact; its scale is 2^-120
constexpr float BIG_ROW = 0x1p100f, SHRINK = 0x1p-64f;
constexpr float ROUND_MAGIC = 12582912.0f;                // 1.5 * 2^23
constexpr float NEAR_HALF = 0.5f - 0x1p-15f;

enum RowKind { ROW_BF16 = 0, ROW_F16 = 1, ROW_F32 = 2, ROW_SWIGLU = 3, ROW_NORM = 4 };

struct RowParams {
  const void* x;                 // rows (norm: the residual, updated in place when delta is given)
  const __nv_bfloat16* delta;    // norm only, may be null
  const float* w;                // norm only
  long long ldx, ldd, ldq, ldo;
  signed char* q;
  float* scale;
  __half* out16;                 // norm only, may be null
  int k, cluster;
  float eps, w_off, inv_k;       // norm only; inv_k = 1 / k
  int* err;
};

// max(|m|, |a|, |b|), NaN if one of them is
VG_DEVINL float max_abs3(float m, float a, float b) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
  return r;
}

// The sum of a norm row's squares has one order whatever form runs the row, where it lies and how many rows there are, so a
// token's codes do not depend on the batch: groups of eight consecutive elements one after the other, blocks of 32 groups
// (256 elements, the lanes of a warp) by a butterfly, blocks i, i + 32, i + 64 .. by lane i, and another butterfly.
constexpr int SUM_BLOCK = 256;
// One butterfly for a warp's MAXC sums: the first steps halve the number of sums a lane carries along with the lanes that
// carry each, so every sum is added in the order of warp_sum. Returns the sum of number `sum_of_lane`.
template <int MAXC>
VG_DEVINL int sum_of_lane(int lane) {
  return MAXC == 1 ? 0 : MAXC == 2 ? lane >> 4 : lane >> 3;
}
template <int MAXC>
VG_DEVINL float warp_sums(float (&s)[MAXC]) {
  static_assert(MAXC == 1 || MAXC == 2 || MAXC == 4, "");
  const int lane = threadIdx.x & 31;
  float v = s[0];
  if constexpr (MAXC == 1) {
    v += __shfl_xor_sync(0xffffffffu, v, 16);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
  } else if constexpr (MAXC == 2) {
    const bool hi = lane & 16;
    v = (hi ? s[1] : s[0]) + __shfl_xor_sync(0xffffffffu, hi ? s[0] : s[1], 16);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
  } else {
    const bool hi = lane & 16, second = lane & 8;
    const float a = (hi ? s[2] : s[0]) + __shfl_xor_sync(0xffffffffu, hi ? s[0] : s[2], 16);
    const float b = (hi ? s[3] : s[1]) + __shfl_xor_sync(0xffffffffu, hi ? s[1] : s[3], 16);
    v = (second ? b : a) + __shfl_xor_sync(0xffffffffu, second ? a : b, 8);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// `blocks` <= 32 * MOST
template <int MOST>
VG_DEVINL float sum_of_blocks(const float* block, int blocks) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const int i = (threadIdx.x & 31) + 32 * j;
    s += i < blocks ? block[i] : 0.f;
  }
  return warp_sum(s);
}

// Over `threads` threads of which this is number `tid`, with one barrier (the block's, or named barrier `bar` of a team): the
// maximum of a non-negative float's bits (so NaN > inf > finite), and (SUM) each warp's MAXC block sums to `block`.
template <bool SUM, int MAXC>
VG_DEVINL void block_reduce(unsigned& mx, float (&ss)[MAXC], unsigned* red_m, float* block, int tid, int threads, int bar = 0) {
  const int lane = tid & 31, w = tid >> 5, nw = threads >> 5;
  mx = __reduce_max_sync(0xffffffffu, mx);
  if constexpr (SUM) {
    const float sum = warp_sums(ss);
    if (lane % (32 / MAXC) == 0) block[w + sum_of_lane<MAXC>(lane) * nw] = sum;
  }
  if (lane == 0) red_m[w] = mx;
  asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(threads) : "memory");
  mx = __reduce_max_sync(0xffffffffu, lane < nw ? red_m[lane] : 0u);
}

VG_DEVINL void unpack8(uint4 a, float* v, bool f16) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (&a.x)[i];
    const float2 f = f16 ? __half22float2(*reinterpret_cast<const __half2*>(&w))
                         : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
VG_DEVINL uint4 pack_bf16(const float* v) {
  uint4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    (&o.x)[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return o;
}
VG_DEVINL uint4 pack_f16_sat(const float* v) {
  uint4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __halves2half2(f32_to_f16_sat(v[2 * i]), f32_to_f16_sat(v[2 * i + 1]));
    (&o.x)[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return o;
}

// What a row's statistics give: the largest value, the scale, the factor from value to code in two terms (the second for
// 16-bit rows only) and (norm) 1 / rms.
struct RowScale {
  float amax, s, f, f_lo, inv;
  bool bad;
};
template <int KIND>
VG_DEVINL RowScale row_scale(const RowParams& p, unsigned mx, float ss) {
  // The norm's factor 1 / rms is common to the row, so the maximum of |res * w| found in the same pass as the sum of
  // squares is enough: one reduction instead of two.
  RowScale o;
  o.inv = KIND == ROW_NORM ? rsqrtf(__fmaf_rn(ss, p.inv_k, p.eps)) : 1.f;
  const float amax = __uint_as_float(mx) * o.inv;
  o.bad = !(amax < INFINITY) || (KIND == ROW_NORM && !(ss < INFINITY));
  o.amax = fmaxf(amax, AMAX_FLOOR);
  o.s = o.bad ? __uint_as_float(0x7fffffffu) : __fdiv_rn(o.amax, INT8_MAX_CODE);       // 2^-120 or more, so 1 / s <= 2^120
  if (KIND == ROW_BF16 || KIND == ROW_F16) {
    if (o.amax > BIG_ROW) o.amax *= SHRINK;                       // so that f_lo does not underflow; the values follow
    o.f = o.bad ? 0.f : __fdiv_rn(INT8_MAX_CODE, o.amax);
    o.f_lo = __fmaf_rn(-o.f, o.amax, INT8_MAX_CODE) * o.f * (1.f / INT8_MAX_CODE);      // exact remainder / amax
  } else {
    o.f = o.bad ? 0.f : __fdiv_rn(1.f, o.s);
    o.f_lo = 0.f;
  }
  return o;
}

// Code of one value: rint(127 v / amax), half to even, decided exactly. v * f is within 127.5 * 2^-23 < 2^-16 of 127 v / amax,
// so the code is the integer next to it or, close to a half, the one beyond the half. Which one, the sign of
// 127 v - half * amax says: both products' leading 24 bits cancel, and what is left of each is exact in fp32 (scaled by a power
// of two, so that nothing leaves its range).
VG_DEVINL uint32_t code_near_half(float v, float f, float amax) {
  const float m = __fmaf_rn(v, f, ROUND_MAGIC), n = m - ROUND_MAGIC, d = __fmaf_rn(v, f, -n);
  if (!(fabsf(d) > NEAR_HALF)) return __float_as_uint(m);
  const float out = copysignf(1.0f, d), half = n + 0.5f * out;    // the neighbour is n + out
  const float unit = amax >= 1.0f ? 0x1p-10f : 0x1p100f, a = amax * unit;
  const float p = half * a, low = __fmaf_rn(half, a, -p);
  const float beyond = out * (__fmaf_rn(INT8_MAX_CODE, v * unit, -p) - low);
  const bool odd = __float_as_uint(m) & 1;
  return __float_as_uint(beyond > 0.f || (beyond == 0.f && odd) ? m + out : m);
}
// Eight values -> eight codes. Adding 1.5 * 2^23 leaves the rounded integer in the low bits of the sum. (cvt.rni runs at an
// eighth of the rate, next to the exponentials.)
// 16-bit rows hold many exact halves (127 v / amax = n + 1/2: one value in 6000 of a Gaussian bf16 row, every second one where
// amax is 254 times a power of two); any other quotient is 2^-20 of its size or more away from a half, since v and amax have
// 11 bits at most. v f + v f_lo, rounded twice, is off by 2^-23 at most, and for a half exactly right: the first product's
// rounding is at most half a step, which the second rounding takes back. (4096 x 17408 bf16: one product 34.4 us, two
// terms 38.3; 4096 x 5120 14.0 and 14.9. A test for halves and a branch, as below: 56, the rows above being the slow ones.)
// fp32 rows can come closer to a half than any such sum: what is near one is decided by code_near_half (4096 x 5120: 20.0
// without, 20.9 with).
template <int KIND>
VG_DEVINL uint2 codes8(const float* v, const RowScale& rs) {
  uint32_t t[8];
  if constexpr (KIND == ROW_BF16 || KIND == ROW_F16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = __float_as_uint(__fadd_rn(__fmaf_rn(v[i], rs.f_lo, __fmul_rn(v[i], rs.f)), ROUND_MAGIC));
  } else if constexpr (KIND == ROW_F32) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float m0 = __fmaf_rn(v[i], rs.f, ROUND_MAGIC), m1 = __fmaf_rn(v[i + 1], rs.f, ROUND_MAGIC);
      t[i] = __float_as_uint(m0);
      t[i + 1] = __float_as_uint(m1);
      most = max_abs3(most, __fmaf_rn(v[i], rs.f, ROUND_MAGIC - m0), __fmaf_rn(v[i + 1], rs.f, ROUND_MAGIC - m1));
    }
    if (most > NEAR_HALF) {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = code_near_half(v[i], rs.f, rs.amax);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = __float_as_uint(__fmaf_rn(v[i], rs.f, ROUND_MAGIC));
  }
  return make_uint2(__byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410));
}
// bf16 rows whose largest value is near the end of the range: see row_scale
template <int KIND, int MAXC>
VG_DEVINL void shrink_big_row(float (&v)[MAXC][8], unsigned mx) {
  if (KIND == ROW_BF16 && __uint_as_float(mx) > BIG_ROW) {
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] *= SHRINK;
  }
}

// Eight elements from element e of a row that starts at `base` and has `limit` of them in memory, as packed words; those
// before `lo` and from `left` on are zero. VEC: 16-byte addresses and whole groups. Else the address may be anything a
// tensor of that type can have: the aligned words around the group are loaded and shifted into place (by the same amount
// in a whole row), as long as they lie inside the row; the edges are read one by one.
template <bool VEC, int ES>
VG_DEVINL void load8_raw(const char* base, long long e, int lo, int left, long long limit, uint32_t* w) {
  constexpr int W = 2 * ES;
  const char* a = base + e * ES;
  if (VEC) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) *reinterpret_cast<uint4*>(w + 4 * i) = *reinterpret_cast<const uint4*>(a + 16 * i);
    return;
  }
  const uint32_t mis = (uint32_t)(reinterpret_cast<uintptr_t>(a) & 15);
  const char* a0 = a - mis;
  if (lo == 0 && left >= 8 && (mis == 0 || (a0 >= base && a0 + W * 4 + 16 <= base + limit * ES))) {
    uint32_t t[W + 4] = {};
#pragma unroll
    for (int i = 0; i < W / 4; ++i) *reinterpret_cast<uint4*>(t + 4 * i) = *reinterpret_cast<const uint4*>(a0 + 16 * i);
    if (mis) *reinterpret_cast<uint4*>(t + W) = *reinterpret_cast<const uint4*>(a0 + W * 4);
    if (mis & 8) {
#pragma unroll
      for (int i = 0; i < W + 2; ++i) t[i] = t[i + 2];
    }
    if (mis & 4) {
#pragma unroll
      for (int i = 0; i < W + 1; ++i) t[i] = t[i + 1];
    }
    if (ES == 2 && (mis & 2)) {
#pragma unroll
      for (int i = 0; i < W; ++i) t[i] = __funnelshift_r(t[i], t[i + 1], 16);
    }
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = t[i];
    return;
  }
  if (ES == 4) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = i >= lo && i < left ? *reinterpret_cast<const uint32_t*>(a + 4 * i) : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint32_t l = i >= lo && i < left ? *reinterpret_cast<const uint16_t*>(a + 2 * i) : 0u;
      const uint32_t h = i + 1 >= lo && i + 1 < left ? *reinterpret_cast<const uint16_t*>(a + 2 * i + 2) : 0u;
      w[i / 2] = l | (h << 16);
    }
  }
}
// Group [e, e + 8) of a row of k 2-byte values, where the row may start anywhere: the 16-byte word at the next boundary takes
// the rest from the next lane; the row's ends and the last lane's part are written one by one. All lanes call this.
VG_DEVINL void store_half_shifted(void* row, int e, int k, uint4 own) {
  uint16_t* dst = static_cast<uint16_t*>(row) + e;
  const uint32_t mis = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15);           // the same in all of the row's groups
  uint32_t t[8] = {own.x, own.y, own.z, own.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) t[4 + i] = __shfl_down_sync(0xffffffffu, t[i], 1);
  if (e >= k) return;
  const int lane = threadIdx.x & 31, head = mis ? (int)(16 - mis) / 2 : 0;          // own values before the boundary
  const bool full = mis ? lane < 31 && e + head + 8 <= k : e + 8 <= k;
  const bool head_done = lane > 0 && e + head <= k;                                 // by the previous lane's word
  if (full) {
    uint32_t s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = t[i];
    if (head & 4) {
#pragma unroll
      for (int i = 0; i < 6; ++i) s[i] = s[i + 2];
    }
    if (head & 2) {
#pragma unroll
      for (int i = 0; i < 5; ++i) s[i] = s[i + 1];
    }
    if (head & 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = __funnelshift_r(s[i], s[i + 1], 16);
    }
    *reinterpret_cast<uint4*>(dst + head) = make_uint4(s[0], s[1], s[2], s[3]);
    if (head_done) return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (!(i < head ? head_done : full) && e + i < k) dst[i] = (uint16_t)(t[i >> 1] >> (16 * (i & 1)));
}
template <bool VEC>
VG_DEVINL void store_codes(signed char* q, int left, uint2 v) {
  if (VEC || (left >= 8 && reinterpret_cast<uintptr_t>(q) % 8 == 0)) {
    *reinterpret_cast<uint2*>(q) = v;
    return;
  }
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) q[i] = (signed char)((&v.x)[i >> 2] >> (8 * (i & 3)));
  }
}
// The codes of group [e, e + 8) of a row of k, where groups start `shift` elements past multiples of eight: the 8-byte
// word at the next multiple takes the rest from the next lane (lane 31 only hands its codes over). What is left at the
// row's ends, and everything when the row of codes is not 8-byte aligned, is written byte by byte. All lanes call this.
VG_DEVINL void store_codes_shifted(signed char* q, int e, int k, int shift, uint2 v) {
  const unsigned long long own = ((unsigned long long)v.y << 32) | v.x;
  const unsigned long long next = __shfl_down_sync(0xffffffffu, own, 1);
  if ((threadIdx.x & 31) == 31 || e >= k) return;
  const bool wide = reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const int word = shift ? e + 8 - shift : e;                        // first multiple of eight inside or after the group's start
  const bool full = wide && word >= 0 && word + 8 <= k;
  const bool lead_done = shift == 0 || (wide && word >= 8 && word <= k);          // by the previous lane's word
  if (full) *reinterpret_cast<unsigned long long*>(q + word) = shift ? (own >> (8 * (8 - shift))) | (next << (8 * shift)) : own;
  if (full && lead_done) return;
  for (int i = 0; i < 8; ++i)
    if (!(i < word - e ? lead_done : full) && e + i >= 0 && e + i < k) q[e + i] = (signed char)(own >> (8 * i));
}

// A row belongs to one CTA, or (CL) to a cluster of them that exchanges its partial statistics through distributed
// shared memory. A thread owns MAXC groups of eight consecutive elements; all its loads are issued before the first use.
// Rows that do not all start on 16-byte boundaries (!VEC) are cut into groups at the boundaries of x (SHIFTED), so x is read
// in whole words whatever the width; the codes are shifted into their own words on the way out, with a lane's
// neighbour supplying the rest. Warps overlap by one group for that: lane 31 repeats the next warp's first. (Bytes stored
// one by one at the seams of warps: 11.7 us at 1237 x 4111, with the overlap 8.7.) The norm keeps the groups of aligned rows,
// which its sum goes by, and reads and writes each from where it is.
template <int KIND, bool VEC, int MAXC, bool CL>
__global__ void __launch_bounds__(1024) row_int8_kernel(const RowParams p) {
  constexpr int ES = KIND == ROW_F32 ? 4 : 2;
  constexpr bool PAIR = KIND == ROW_SWIGLU || KIND == ROW_NORM;
  constexpr bool SHIFTED = !VEC && KIND != ROW_NORM;
  __shared__ unsigned red_m[32];
  __shared__ unsigned peer[MAX_CLUSTER];
  __shared__ float block[KIND != ROW_NORM ? 1 : CL ? ROW_MAX / SUM_BLOCK : 32 * MAXC];
  pdl_trigger();
  if (CL) cluster_arrive_relaxed();
  pdl_wait();
  const int rank = CL ? (int)cluster_ctarank() : 0;
  const int nrank = CL ? p.cluster : 1;
  const size_t row = CL ? blockIdx.x / nrank : blockIdx.x;
  const int T = blockDim.x * nrank;
  const int tid = threadIdx.x + rank * blockDim.x;
  const int k = p.k;
  char* x_row = static_cast<char*>(const_cast<void*>(p.x)) + row * p.ldx * ES;
  const char* d_row = reinterpret_cast<const char*>(p.delta + row * p.ldd);
  constexpr int LANES = SHIFTED ? 31 : 32;                         // groups of its own that a warp has
  const int shift = !SHIFTED ? 0 : (int)((16 - (reinterpret_cast<uintptr_t>(x_row) & 15)) & 15) / ES;
  const int e0 = ((tid >> 5) * LANES + (tid & 31)) * 8 - ((8 - shift) & 7), e_step = T / 32 * LANES * 8;
  const bool owner = !SHIFTED || (tid & 31) < 31;
  uint32_t xr[MAXC][2 * ES], yr[MAXC][4];
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    const int e = e0 + c * e_step, lo = max(0, -e);
    if (e < k) {
      load8_raw<VEC, ES>(x_row, e, lo, k - e, KIND == ROW_SWIGLU ? 2 * k : k, xr[c]);
      if (KIND == ROW_SWIGLU) load8_raw<VEC, 2>(x_row, k + e, lo, k - e, 2 * k, yr[c]);
      if (KIND == ROW_NORM && p.delta) load8_raw<VEC, 2>(d_row, e, lo, k - e, k, yr[c]);
    }
  }
  float v[MAXC][8];
  float amax = 0.f, ss[MAXC] = {};
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    const int e = e0 + c * e_step, lo = max(0, -e);
    if (e < k) {
      if (ES == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = __uint_as_float(xr[c][i]);
      } else {
        unpack8(make_uint4(xr[c][0], xr[c][1], xr[c][2], xr[c][3]), v[c], KIND == ROW_F16);
      }
      float y[8];
      if (PAIR) unpack8(make_uint4(yr[c][0], yr[c][1], yr[c][2], yr[c][3]), y, false);
      if (KIND == ROW_SWIGLU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = silu(v[c][i]) * y[i];
      }
      if (KIND == ROW_NORM) {
        if (p.delta) {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] += v[c][i];
          const uint4 r4 = pack_bf16(y);
          xr[c][0] = r4.x; xr[c][1] = r4.y; xr[c][2] = r4.z; xr[c][3] = r4.w;      // stored after the reduction
          unpack8(r4, v[c], false);
        }
        uint32_t ww[8];
        load8_raw<VEC, 4>(reinterpret_cast<const char*>(p.w), e, lo, k - e, k, ww);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss[c] = __fmaf_rn(v[c][i], v[c][i], ss[c]);
          v[c][i] *= __uint_as_float(ww[i]) + p.w_off;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) amax = max_abs3(amax, v[c][i], v[c][i + 1]);
  }
  unsigned mx = __float_as_uint(amax);
  block_reduce<KIND == ROW_NORM && !CL>(mx, ss, red_m, block, threadIdx.x, blockDim.x);
  if (CL) {
    float warps = 0.f;
    if constexpr (KIND == ROW_NORM) warps = warp_sums(ss);
    cluster_wait();                                   // every CTA of the row has started
    if ((int)threadIdx.x < nrank) dsmem_st_u32(dsmem_map(smem_u32(&peer[rank]), threadIdx.x), mx);
    if constexpr (KIND == ROW_NORM) {                 // each of the lanes that have a sum tells one rank
      const int lane = tid & 31, to = lane % (32 / MAXC);
      if (to < nrank) dsmem_st_f32(dsmem_map(smem_u32(&block[(tid >> 5) + sum_of_lane<MAXC>(lane) * (T >> 5)]), to), warps);
    }
    cluster_sync_all();
    mx = 0;
    for (int r = 0; r < nrank; ++r) mx = max(mx, peer[r]);
  }
  float sum = 0.f;
  if constexpr (KIND == ROW_NORM) {
    const int blocks = (k + SUM_BLOCK - 1) / SUM_BLOCK;
    if (CL && blocks > 128) sum = sum_of_blocks<ROW_MAX / SUM_BLOCK / 32>(block, blocks);
    else sum = sum_of_blocks<CL ? 4 : MAXC>(block, blocks);
  }

  const RowScale rs = row_scale<KIND>(p, mx, sum);
  shrink_big_row<KIND>(v, mx);
  if (tid == 0) p.scale[row] = rs.s;
  if (KIND == ROW_NORM) {
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] *= rs.inv;
  }
  const uint4 nan4 = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    const int e = e0 + c * e_step;
    const uint2 codes = rs.bad ? make_uint2(0u, 0u) : codes8<KIND>(v[c], rs);
    if (SHIFTED) store_codes_shifted(p.q + row * p.ldq, e, k, shift, codes);
    if (e < k && owner) {
      if (!SHIFTED) store_codes<VEC>(p.q + row * p.ldq + e, k - e, codes);
    }
    if constexpr (KIND == ROW_NORM) {
      const uint4 r4 = make_uint4(xr[c][0], xr[c][1], xr[c][2], xr[c][3]);
      if (VEC && e < k) {
        if (p.delta) *reinterpret_cast<uint4*>(x_row + (long long)e * 2) = r4;
        if (p.out16) *reinterpret_cast<uint4*>(p.out16 + row * p.ldo + e) = rs.bad ? nan4 : pack_f16_sat(v[c]);
      }
      if (!VEC) {
        if (p.delta) store_half_shifted(x_row, e, k, r4);
        if (p.out16) store_half_shifted(p.out16 + row * p.ldo, e, k, rs.bad ? nan4 : pack_f16_sat(v[c]));
      }
    }
  }
}

// Many rows: persistent blocks with a ring of whole rows in shared memory, filled by bulk copies several rows ahead, so
// the memory system stays busy while a block reduces, quantises and stores. A row's slot is refilled as soon as the
// reduction's barrier has shown that every thread holds its part in registers: one barrier per row.
// Rows so wide that an SM holds a single block: TEAMS = 2 halves of the block take turns on the rows of one ring, so one
// half computes while the other waits for its row or its barrier (4096 x 17408 SwiGLU: 71 -> 57 us). A slot of an odd ring
// passes from one team to the other, so a team may come to a slot whose previous row has not even landed (copies may land
// out of order); the one-bit parity of its barrier cannot tell that phase from the one waited for. `filled` can: it names
// the row whose copy was last issued into the slot, and a team looks at the barrier only once its own row is there.
template <int KIND, int MAXC, int TEAMS>
__global__ void __launch_bounds__(TEAMS == 2 ? 1024 : MAXC == 4 ? 640 : 1024, MAXC == 4 && KIND != ROW_NORM ? 2 : 1)
row_int8_ring_kernel(const RowParams p, int n, int slots, int slot_bytes) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[RING_SLOTS];
  __shared__ unsigned red_m[TEAMS][2][32];
  __shared__ float block[2][KIND != ROW_NORM ? 1 : RING_GROUPS / 32];
  __shared__ int stuck[TEAMS];
  __shared__ volatile int filled[RING_SLOTS];
  constexpr int ES = KIND == ROW_F32 ? 4 : 2;
  pdl_trigger();
  const int k = p.k, T = blockDim.x / TEAMS, step = gridDim.x;
  const int team = TEAMS == 1 ? 0 : (int)threadIdx.x / T, tid = threadIdx.x - team * T;
  const uint32_t x_bytes = (uint32_t)k * ES * (KIND == ROW_SWIGLU ? 2 : 1);
  const bool two = KIND == ROW_NORM && p.delta;
  if (threadIdx.x == 0) {
    for (int i = 0; i < slots; ++i) {
      mbar_init(full + i, 1);
      filled[i] = -1;
    }
    for (int i = 0; i < TEAMS; ++i) stuck[i] = 0;
    fence_mbar_init();
  }
  __syncthreads();
  auto fill = [&](int slot, int j, size_t row) {
    uint8_t* dst = ring + (size_t)slot * slot_bytes;
    mbar_arrive_expect_tx(full + slot, two ? 2 * x_bytes : x_bytes);
    tma_bulk_g2s(dst, static_cast<const char*>(p.x) + row * p.ldx * ES, x_bytes, full + slot);
    if (two) tma_bulk_g2s(dst + x_bytes, p.delta + row * p.ldd, x_bytes, full + slot);
    if (TEAMS > 1) {
      __threadfence_block();
      filled[slot] = j;
    }
  };
  pdl_wait();
  if (threadIdx.x == 0)
    for (int i = 0; i < slots && (int)blockIdx.x + i * step < n; ++i) fill(i, i, blockIdx.x + (size_t)i * step);
  // the block's rows are blockIdx.x + j * step in slots j % slots; a team takes every TEAMS-th of them
  int slot = team, it = 0;
  uint32_t ph = 0;
  for (long long row = blockIdx.x + (long long)team * step; row < n; row += (long long)TEAMS * step, ++it) {
    const int j = it * TEAMS + team;
    bool ok = true;
    if (TEAMS > 1) {
      const uint64_t t0 = global_ns();
      while (filled[slot] != j && ok) ok = global_ns() - t0 < 200ull * 1000 * 1000;
      __threadfence_block();
    }
    if (!ok || !mbar_wait(full + slot, ph)) {
      if (p.err) atomicCAS(p.err, 0, (int)VG_ERR_TMA_WAIT);
      stuck[team] = 1;
    }
    const uint8_t* src = ring + (size_t)slot * slot_bytes;
    float v[MAXC][8];
    float amax = 0.f, ss[MAXC] = {};
#pragma unroll
    for (int c = 0; c < MAXC; ++c) {
      const int e = (tid + c * T) * 8;
      if (e < k) {
        if (KIND == ROW_F32) {
          *reinterpret_cast<float4*>(v[c]) = *reinterpret_cast<const float4*>(src + (size_t)e * 4);
          *reinterpret_cast<float4*>(v[c] + 4) = *reinterpret_cast<const float4*>(src + (size_t)e * 4 + 16);
        } else {
          unpack8(*reinterpret_cast<const uint4*>(src + (size_t)e * 2), v[c], KIND == ROW_F16);
        }
        if (KIND == ROW_SWIGLU) {
          float u[8];
          unpack8(*reinterpret_cast<const uint4*>(src + (size_t)(k + e) * 2), u, false);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] = silu(v[c][i]) * u[i];
        }
        if (two) {
          float d[8];
          unpack8(*reinterpret_cast<const uint4*>(src + x_bytes + (size_t)e * 2), d, false);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] += v[c][i];
          const uint4 r4 = pack_bf16(d);
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(const_cast<void*>(p.x)) + row * p.ldx + e) = r4;
          unpack8(r4, v[c], false);
        }
        if (KIND == ROW_NORM) {
          const float4 w0 = *reinterpret_cast<const float4*>(p.w + e), w1 = *reinterpret_cast<const float4*>(p.w + e + 4);
          const float ww[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ss[c] = __fmaf_rn(v[c][i], v[c][i], ss[c]);
            v[c][i] *= ww[i] + p.w_off;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; i += 2) amax = max_abs3(amax, v[c][i], v[c][i + 1]);
    }
    unsigned mx = __float_as_uint(amax);
    block_reduce<KIND == ROW_NORM>(mx, ss, red_m[team][it & 1], block[it & 1], tid, T, team + 1);
    if (stuck[team]) break;                                // seen by the whole team: set before the barrier
    if (tid == 0 && row + (long long)slots * step < n) fill(slot, j + slots, row + (size_t)slots * step);
    float sum = 0.f;
    if constexpr (KIND == ROW_NORM)
      sum = sum_of_blocks<MAXC == 4 ? (RING_GROUPS / 32 + 31) / 32 : 1>(block[it & 1], (k + SUM_BLOCK - 1) / SUM_BLOCK);
    const RowScale rs = row_scale<KIND>(p, mx, sum);
    shrink_big_row<KIND>(v, mx);
    if (tid == 0) p.scale[row] = rs.s;
#pragma unroll
    for (int c = 0; c < MAXC; ++c) {
      const int e = (tid + c * T) * 8;
      if (e < k) {
        if (KIND == ROW_NORM) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] *= rs.inv;
        }
        *reinterpret_cast<uint2*>(p.q + (size_t)row * p.ldq + e) = rs.bad ? make_uint2(0u, 0u) : codes8<KIND>(v[c], rs);
        if (KIND == ROW_NORM && p.out16) {
          const uint4 nan4 = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
          *reinterpret_cast<uint4*>(p.out16 + (size_t)row * p.ldo + e) = rs.bad ? nan4 : pack_f16_sat(v[c]);
        }
      }
    }
    slot += TEAMS;
    if (slot >= slots) { slot -= slots; ph ^= 1; }
  }
  if (stuck[team] && tid == 0)
    for (int i = 0; i < 64; ++i) __nanosleep(1000);        // let copies in flight land before the block ends
}

template <typename OUT>
VG_DEVINL OUT from_f32(float v);
template <> VG_DEVINL float from_f32<float>(float v) { return v; }
template <> VG_DEVINL __half from_f32<__half>(float v) { return v != v ? __ushort_as_half(0x7fff) : f32_to_f16_sat(v); }
template <> VG_DEVINL __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Read-back, eight codes per thread and row, R rows per block so that R loads are in flight. (Sixteen per thread leave two
// 16-byte stores 32 bytes apart per lane: 15.8 us instead of 10.8 at 4096 x 5120.)
template <typename OUT>
VG_DEVINL void dequant4(uint32_t c, float s, OUT* o) {
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = from_f32<OUT>((float)(signed char)(c >> (8 * i)) * s);
}
template <typename OUT, int R>
__global__ void __launch_bounds__(1024) dequant_int8_kernel(const signed char* q, long long ldq,
                                                            const float* scale, OUT* out,
                                                            long long ldo, int n, int k) {
  pdl_trigger();
  pdl_wait();
  const long long row0 = (long long)blockIdx.x * R;
  const int e = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  if (e >= k) return;
  uint2 c[R];
  float s[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (R > 1 && row0 + r >= n) break;
    c[r] = *reinterpret_cast<const uint2*>(q + (row0 + r) * ldq + e);
    s[r] = scale[row0 + r];
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (R > 1 && row0 + r >= n) break;
    alignas(16) OUT o[8];
    dequant4(c[r].x, s[r], o);
    dequant4(c[r].y, s[r], o + 4);
    OUT* dst = out + (row0 + r) * ldo + e;
#pragma unroll
    for (int i = 0; i < (int)sizeof(OUT) / 2; ++i) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(o)[i];
  }
}

// Any width and pitch: groups of eight that start on the output's 16-byte boundaries; their codes come from the two
// aligned words around them where those lie inside the row.
template <typename OUT>
__global__ void __launch_bounds__(256) dequant_int8_loose_kernel(const signed char* q, long long ldq,
                                                                 const float* scale, OUT* out,
                                                                 long long ldo, int k) {
  pdl_trigger();
  pdl_wait();
  const size_t row = blockIdx.x;
  const float s = scale[row];
  const signed char* src = q + row * ldq;
  OUT* dst = out + row * ldo;
  const int head = (int)((16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15) / (int)sizeof(OUT);   // elements before the first boundary
  for (int g = blockIdx.y * blockDim.x + threadIdx.x;; g += gridDim.y * blockDim.x) {
    const int e = head + (g - 1) * 8;
    if (e >= k) break;
    const uint32_t mis = (uint32_t)(reinterpret_cast<uintptr_t>(src + e) & 7);
    const signed char* a0 = src + e - (int)mis;
    if (e >= 0 && e + 8 <= k && (mis == 0 || (a0 >= src && a0 + 16 <= src + k))) {
      unsigned long long w = *reinterpret_cast<const unsigned long long*>(a0);
      if (mis) w = (w >> (8 * mis)) | (*reinterpret_cast<const unsigned long long*>(a0 + 8) << (64 - 8 * mis));
      alignas(16) OUT o[8];
      dequant4((uint32_t)w, s, o);
      dequant4((uint32_t)(w >> 32), s, o + 4);
#pragma unroll
      for (int i = 0; i < (int)sizeof(OUT) / 2; ++i) reinterpret_cast<uint4*>(dst + e)[i] = reinterpret_cast<const uint4*>(o)[i];
    } else {
      for (int i = max(0, -e); i < 8 && e + i < k; ++i) dst[e + i] = from_f32<OUT>((float)src[e + i] * s);
    }
  }
}

// Ring of all blocks of an SM. More of it leaves too little L1 for the norm's weights (4096 x 17408: 89 us with 200 KB, 94
// with 212); two teams without weights want a third slot.
constexpr int RING_BYTES = 200 * 1024, RING_TEAM_BYTES = 212 * 1024;
constexpr int RING_PER_SM = 16;                   // blocks per SM
// Rows per SM from which the ring form is taken, by row width in groups (us: row form / ring form):
//   up to 1024   quantise 5120: 1184 rows 6.5 / 6.8, 1500 8.1 / 7.4, 4096 18.2 / 14.9; norm 5120: 1184 11.8 / 12.5, 2000 17.6 /
//                18.1, 4096 31.2 / 29.2; SwiGLU 8192: 1184 11.8 / 11.7, 4096 33.3 / 31.0. Below about 3000 elements the row
//                form is still ahead (norm 2560, 4096 rows: 16.3 / 19.5).
//   up to 1280   all but the norm: SwiGLU 8704: 600 rows 7.6 / 10.4, 3000 26.6 / 27.2; quantise 8704: 1000 8.6 / 9.6, 3000
//                21.2 / 21.3, 4096 28.3 / 25.1. Norm 8704: 600 14.2 / 14.0, 4096 74.7 / 57.7.
//   wider        SwiGLU 17408: 149 rows 6.5 / 6.8, 296 9.0 / 8.5, 333 10.6 / 10.3, 1000 25.6 / 18.2, 4096 96 / 57; 12800: 149
//                5.4 / 6.1, 600 12.6 / 11.3; quantise 17408: 149 5.4 / 5.0, 4096 77 / 38; norm 17408: 149 11.9 / 9.8, 4096 204 / 90.
constexpr int RING_MIN_ROWS = 8, RING_MIN_MID = 20, RING_MIN_WIDE = 1;
constexpr int RING_MID_GROUPS = 1280;

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  n = known[dev & 63].load();
  if (n <= 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) known[dev & 63].store(n);
  return n;
}

template <int KIND, bool VEC>
cudaError_t launch_shape(RowParams p, int n, cudaStream_t st) {
  // shifted rows may begin and end inside a group, and a warp has 31 of its own
  constexpr bool SHIFTED = !VEC && KIND != ROW_NORM;
  const int groups = SHIFTED ? (p.k + 14) / 8 : (p.k + 7) / 8;
  constexpr int lanes = SHIFTED ? 31 : 32;
  auto threads = [&](int parts) { return dim3((groups + parts * lanes - 1) / (parts * lanes) * 32); };
  p.cluster = 1;
  // Many shifted 16-bit rows without a second input: two groups a thread halve the fixed instructions. 592 x 4111 6.0 -> 5.0 us,
  // 1237 9.2 -> 8.4, 4096 26.7 -> 22.7 (but 800 6.6 -> 7.5); 300 x 4111 3.2 -> 4.2, 4096 x 2051 12.7 -> 14.0, fp32 rows 25.3 -> 26.6.
  const bool two = SHIFTED && KIND <= ROW_F16 && groups > 16 * lanes && n >= 4 * sm_count();
  if (groups <= 32 * lanes && !two) return launch_pdl(row_int8_kernel<KIND, VEC, 1, false>, dim3(n), threads(1), 0, st, p);
  if (groups <= 64 * lanes) return launch_pdl(row_int8_kernel<KIND, VEC, 2, false>, dim3(n), threads(2), 0, st, p);
  while (p.cluster < MAX_CLUSTER && p.cluster * 64 * lanes < groups) p.cluster *= 2;
  if constexpr (SHIFTED) {
    if (groups > p.cluster * 64 * lanes)
      return launch_pdl_cluster(row_int8_kernel<KIND, false, 3, true>, dim3(n * p.cluster), threads(3 * p.cluster), p.cluster, 0, st, p);
  }
  return launch_pdl_cluster(row_int8_kernel<KIND, VEC, 2, true>, dim3(n * p.cluster), threads(2 * p.cluster), p.cluster, 0, st, p);
}

template <int KIND, int MAXC, int TEAMS>
int launch_ring(const RowParams& p, int n, int slot_bytes, int sms, cudaStream_t st) {
  constexpr int BYTES = TEAMS == 2 ? RING_TEAM_BYTES : RING_BYTES;
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (!(done.load() & (1ull << (dev & 63)))) {
    e = cudaFuncSetAttribute(row_int8_ring_kernel<KIND, MAXC, TEAMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    if (e != cudaSuccess) return (int)e;
    done.fetch_or(1ull << (dev & 63));
  }
  const int groups = p.k / 8, threads = ((groups + MAXC - 1) / MAXC + 31) / 32 * 32;
  const int room = BYTES / slot_bytes;        // slots an SM holds
  const int per_sm = TEAMS == 2 ? 1 : max(1, min(min(RING_PER_SM, 2048 / threads), max(room / 3, min(2, room / 2))));
  const int slots = max(2, min(RING_SLOTS, BYTES / per_sm / slot_bytes));
  const int grid = min(n, sms * per_sm);
  return (int)launch_pdl(row_int8_ring_kernel<KIND, MAXC, TEAMS>, dim3(grid), dim3(threads * TEAMS), (size_t)slots * slot_bytes, st, p, n, slots, slot_bytes);
}

// `esize`: bytes of one input element; VEC wants whole groups of eight and 16-byte addresses on every row
template <int KIND>
int launch_row(const RowParams& p, int n, int esize, cudaStream_t st) {
  if (p.k <= 0 || p.k > ROW_MAX || n < 0 || n > (1 << 27)) return -2;
  if (n == 0) return 0;
  bool vec = p.k % 8 == 0 && aligned(p.x, 16) && (n == 1 || (p.ldx * esize) % 16 == 0) && aligned(p.q, 8) &&
             (n == 1 || p.ldq % 8 == 0);
  if (KIND == ROW_NORM) {
    vec = vec && aligned(p.w, 16);
    if (p.delta) vec = vec && aligned(p.delta, 16) && (n == 1 || p.ldd % 8 == 0);
    if (p.out16) vec = vec && aligned(p.out16, 16) && (n == 1 || p.ldo % 8 == 0);
  }
  const int sms = sm_count(), slot = p.k * esize * ((KIND == ROW_SWIGLU || p.delta) ? 2 : 1), groups = p.k / 8;
  const int ring_rows = groups <= 1024 ? RING_MIN_ROWS
                        : KIND != ROW_NORM && groups <= RING_MID_GROUPS ? RING_MIN_MID : RING_MIN_WIDE;
  if (vec && n >= ring_rows * sms && slot % 16 == 0 && 2 * slot <= RING_BYTES && groups <= RING_GROUPS) {
    if constexpr (KIND == ROW_SWIGLU) {
      if (4 * slot > RING_BYTES && groups > 1024) return launch_ring<KIND, 5, 2>(p, n, slot, sms, st);
    }
    return groups <= 32 ? launch_ring<KIND, 1, 1>(p, n, slot, sms, st)
           : groups <= 1024 ? launch_ring<KIND, 2, 1>(p, n, slot, sms, st)
                            : launch_ring<KIND, 4, 1>(p, n, slot, sms, st);
  }
  const cudaError_t e = vec ? launch_shape<KIND, true>(p, n, st) : launch_shape<KIND, false>(p, n, st);
  return (int)e;
}

template <typename OUT>
int launch_dequant(const signed char* q, long long ldq, const float* scale, void* out, long long ldo, int n, int k,
                   cudaStream_t st) {
  const bool vec = k % 8 == 0 && aligned(q, 8) && aligned(out, 16) && (n == 1 || (ldq % 8 == 0 && (ldo * sizeof(OUT)) % 16 == 0));
  OUT* o = static_cast<OUT*>(out);
  if (!vec)
    return (int)launch_pdl(dequant_int8_loose_kernel<OUT>, dim3(n, min((k / 8 + 2 + 255) / 256, 64)), dim3(256), 0, st, q, ldq, scale,
                           o, ldo, k);
  const int words = k / 8, ny = (words + 1023) / 1024, threads = ((words + ny - 1) / ny + 31) / 32 * 32;
  if (n >= 512) return (int)launch_pdl(dequant_int8_kernel<OUT, 4>, dim3((n + 3) / 4, ny), dim3(threads), 0, st, q, ldq, scale, o, ldo, n, k);
  return (int)launch_pdl(dequant_int8_kernel<OUT, 1>, dim3(n, ny), dim3(threads), 0, st, q, ldq, scale, o, ldo, n, k);
}
}  // namespace

extern "C" int vg_quant_int8(const void* x, long long ldx, int dtype, int n, int k, void* q, long long ldq, float* scale,
                             int* err, cudaStream_t st) {
  RowParams p{};
  p.x = x; p.ldx = ldx; p.k = k; p.q = static_cast<signed char*>(q); p.ldq = ldq; p.scale = scale; p.err = err;
  switch (dtype) {
    case ROW_BF16: return launch_row<ROW_BF16>(p, n, 2, st);
    case ROW_F16: return launch_row<ROW_F16>(p, n, 2, st);
    case ROW_F32: return launch_row<ROW_F32>(p, n, 4, st);
  }
  return -2;
}

extern "C" int vg_swiglu_int8(const void* gu, long long ldx, int n, int inter, void* q, long long ldq, float* scale,
                              int* err, cudaStream_t st) {
  RowParams p{};
  p.x = gu; p.ldx = ldx; p.k = inter; p.q = static_cast<signed char*>(q); p.ldq = ldq; p.scale = scale; p.err = err;
  return launch_row<ROW_SWIGLU>(p, n, 2, st);
}

extern "C" int vg_add_rmsnorm_int8(void* res, long long ld_res, const void* delta, long long ld_delta, const float* w, int n,
                                   int h, float eps, int plus_one, void* q, long long ldq, float* scale, void* out16,
                                   long long ld_out16, int* err, cudaStream_t st) {
  RowParams p{};
  p.x = res; p.ldx = ld_res; p.delta = static_cast<const __nv_bfloat16*>(delta); p.ldd = ld_delta; p.w = w; p.k = h;
  p.eps = eps; p.inv_k = h > 0 ? 1.0f / (float)h : 0.f; p.w_off = plus_one ? 1.0f : 0.0f; p.q = static_cast<signed char*>(q); p.ldq = ldq; p.scale = scale; p.err = err;
  p.out16 = static_cast<__half*>(out16); p.ldo = ld_out16;
  return launch_row<ROW_NORM>(p, n, 2, st);
}

extern "C" int vg_dequant_int8(const void* q, long long ldq, const float* scale, void* out, long long ldo, int dtype, int n,
                               int k, int*, cudaStream_t st) {
  if (k <= 0 || n < 0) return -2;
  if (n == 0) return 0;
  const signed char* c = static_cast<const signed char*>(q);
  switch (dtype) {
    case ROW_BF16: return launch_dequant<__nv_bfloat16>(c, ldq, scale, out, ldo, n, k, st);
    case ROW_F16: return launch_dequant<__half>(c, ldq, scale, out, ldo, n, k, st);
    case ROW_F32: return launch_dequant<float>(c, ldq, scale, out, ldo, n, k, st);
  }
  return -2;
}
