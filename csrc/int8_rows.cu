// Row quantisers of the 8-bit integer (W8A8) path: one scale per token, symmetric codes.
//
//   s = max(max_k |y_k| / 127, 2^-120),   q_k = rint(y_k / s)   (half to even, |q| <= 127)
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
#include "common.cuh"
#include "api.h"

namespace {
using namespace vg;

constexpr int MAX_CLUSTER = 8;
constexpr float INT8_MAX_CODE = 127.0f;
constexpr float SCALE_FLOOR = 7.52316384526264e-37f;      // 2^-120

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
  float eps, w_off;
};

VG_DEVINL void dsmem_st_f32x2(uint32_t addr, float a, float b) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}

// Block-wide maximum of a non-negative float's bits (so NaN > inf > finite) and sum, one barrier.
template <bool SUM>
VG_DEVINL void block_reduce(unsigned& mx, float& sum, unsigned* red_m, float* red_s) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  mx = __reduce_max_sync(0xffffffffu, mx);
  if (SUM) sum = warp_sum(sum);
  if (lane == 0) {
    red_m[w] = mx;
    if (SUM) red_s[w] = sum;
  }
  __syncthreads();
  mx = __reduce_max_sync(0xffffffffu, lane < nw ? red_m[lane] : 0u);
  if (SUM) sum = warp_sum(lane < nw ? red_s[lane] : 0.f);
}

template <int KIND>
VG_DEVINL float load_one(const RowParams& p, size_t row, int e) {
  if (KIND == ROW_F32) return static_cast<const float*>(p.x)[row * p.ldx + e];
  if (KIND == ROW_F16) return __half2float(static_cast<const __half*>(p.x)[row * p.ldx + e]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p.x)[row * p.ldx + e]);
}

template <int KIND>
VG_DEVINL void load_eight(const RowParams& p, size_t row, int e, float* v) {
  if (KIND == ROW_F32) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p.x) + row * p.ldx + e);
    const float4 a = s[0], b = s[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else if (KIND == ROW_F16) {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p.x) + row * p.ldx + e);
    const __half2* h = reinterpret_cast<const __half2*>(&a);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.x) + row * p.ldx + e);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

// A row belongs to one CTA, or (CL) to a cluster of them that exchanges its partial statistics through distributed
// shared memory. A thread owns MAXC groups of eight elements: consecutive ones with 16-byte accesses (VEC), or strided
// by all the row's threads with single accesses where the width or an address does not allow that.
template <int KIND, bool VEC, int MAXC, bool CL>
__global__ void __launch_bounds__(1024) row_int8_kernel(const RowParams p) {
  __shared__ unsigned red_m[32];
  __shared__ float red_s[32];
  __shared__ float2 peer[MAX_CLUSTER];
  pdl_trigger();
  if (CL) cluster_arrive_relaxed();
  pdl_wait();
  const int rank = CL ? (int)cluster_ctarank() : 0;
  const int nrank = CL ? p.cluster : 1;
  const size_t row = CL ? blockIdx.x / nrank : blockIdx.x;
  const int T = blockDim.x * nrank;
  const int tid = threadIdx.x + rank * blockDim.x;
  const int k = p.k;
  float v[MAXC][8];
  unsigned mx = 0;
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    if (VEC) {
      const int e = (tid + c * T) * 8;
      if (e < k) {
        load_eight<KIND>(p, row, e, v[c]);
        if (KIND == ROW_SWIGLU) {
          float u[8];
          load_eight<KIND>(p, row, k + e, u);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] = silu(v[c][i]) * u[i];
        }
        if (KIND == ROW_NORM && p.delta) {
          const uint4 d4 = *reinterpret_cast<const uint4*>(p.delta + row * p.ldd + e);
          const __nv_bfloat16* d = reinterpret_cast<const __nv_bfloat16*>(&d4);
          uint4 r4;
          __nv_bfloat16* r = reinterpret_cast<__nv_bfloat16*>(&r4);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            r[i] = __float2bfloat16_rn(v[c][i] + __bfloat162float(d[i]));
            v[c][i] = __bfloat162float(r[i]);
          }
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(const_cast<void*>(p.x)) + row * p.ldx + e) = r4;
        }
        if (KIND == ROW_NORM) {
          const float4 w0 = *reinterpret_cast<const float4*>(p.w + e), w1 = *reinterpret_cast<const float4*>(p.w + e + 4);
          const float ww[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ss += v[c][i] * v[c][i];
            v[c][i] *= ww[i] + p.w_off;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = tid + (c * 8 + i) * T;
        float y = 0.f;
        if (e < k) {
          y = load_one<KIND>(p, row, e);
          if (KIND == ROW_SWIGLU) y = silu(y) * load_one<KIND>(p, row, k + e);
          if (KIND == ROW_NORM) {
            if (p.delta) {
              const __nv_bfloat16 r = __float2bfloat16_rn(y + __bfloat162float(p.delta[row * p.ldd + e]));
              static_cast<__nv_bfloat16*>(const_cast<void*>(p.x))[row * p.ldx + e] = r;
              y = __bfloat162float(r);
            }
            ss += y * y;
            y *= p.w[e] + p.w_off;
          }
        }
        v[c][i] = y;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(v[c][i]) & 0x7fffffffu);
  }
  block_reduce<KIND == ROW_NORM>(mx, ss, red_m, red_s);
  if (CL) {
    cluster_wait();                                   // every CTA of the row has started
    if ((int)threadIdx.x < nrank) dsmem_st_f32x2(dsmem_map(smem_u32(&peer[rank]), threadIdx.x), __uint_as_float(mx), ss);
    cluster_sync_all();
    mx = 0;
    ss = 0.f;
    for (int r = 0; r < nrank; ++r) {                 // rank order: the sum does not depend on timing
      mx = max(mx, __float_as_uint(peer[r].x));
      ss += peer[r].y;
    }
  }

  // The norm's factor 1 / rms is common to the row, so the maximum of |res * w| found in the same pass as the sum of
  // squares is enough: one reduction instead of two.
  const float amax = __uint_as_float(mx);
  float inv = 1.f;
  bool bad = mx >= 0x7f800000u;
  if (KIND == ROW_NORM) {
    bad |= !(ss < INFINITY);
    inv = rsqrtf(ss / (float)k + p.eps);
  }
  const float s = bad ? __uint_as_float(0x7fffffffu) : fmaxf(__fdiv_rn(amax * inv, INT8_MAX_CODE), SCALE_FLOOR);
  // rint(y * (inv / s)): |y| * inv / s <= 127 (1 + 2^-22), which rounds to 127 at most
  const float f = bad ? 0.f : __fdiv_rn(inv, s);
  if (tid == 0) p.scale[row] = s;
  signed char* q = p.q + row * p.ldq;
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    if (VEC) {
      const int e = (tid + c * T) * 8;
      if (e < k) {
        uint2 o;
        unsigned* ow = reinterpret_cast<unsigned*>(&o);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          int b[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) b[i] = bad ? 0 : __float2int_rn(v[c][4 * j + i] * f);
          ow[j] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        }
        *reinterpret_cast<uint2*>(q + e) = o;
        if (KIND == ROW_NORM && p.out16) {
          uint4 h4;
          __half* h = reinterpret_cast<__half*>(&h4);
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = bad ? __ushort_as_half(0x7fff) : f32_to_f16_sat(v[c][i] * inv);
          *reinterpret_cast<uint4*>(p.out16 + row * p.ldo + e) = h4;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = tid + (c * 8 + i) * T;
        if (e < k) {
          q[e] = (signed char)(bad ? 0 : __float2int_rn(v[c][i] * f));
          if (KIND == ROW_NORM && p.out16)
            p.out16[row * p.ldo + e] = bad ? __ushort_as_half(0x7fff) : f32_to_f16_sat(v[c][i] * inv);
        }
      }
    }
  }
}

template <typename OUT>
VG_DEVINL OUT from_f32(float v);
template <> VG_DEVINL float from_f32<float>(float v) { return v; }
template <> VG_DEVINL __half from_f32<__half>(float v) { return v != v ? __ushort_as_half(0x7fff) : f32_to_f16_sat(v); }
template <> VG_DEVINL __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight codes per thread where the width and the addresses allow wide accesses, else one.
template <typename OUT, bool VEC>
__global__ void __launch_bounds__(256) dequant_int8_kernel(const signed char* __restrict__ q, long long ldq,
                                                           const float* __restrict__ scale, OUT* __restrict__ out,
                                                           long long ldo, int k) {
  pdl_trigger();
  pdl_wait();
  const size_t row = blockIdx.x;
  const float s = scale[row];
  const signed char* src = q + row * ldq;
  OUT* dst = out + row * ldo;
  constexpr int W = VEC ? 8 : 1;
  for (int e = (blockIdx.y * blockDim.x + threadIdx.x) * W; e < k; e += gridDim.y * blockDim.x * W) {
    if (VEC) {
      const uint2 c2 = *reinterpret_cast<const uint2*>(src + e);
      const signed char* c = reinterpret_cast<const signed char*>(&c2);
      alignas(16) OUT o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = from_f32<OUT>((float)c[i] * s);
#pragma unroll
      for (int i = 0; i < (int)sizeof(OUT) / 2; ++i) reinterpret_cast<uint4*>(dst + e)[i] = reinterpret_cast<const uint4*>(o)[i];
    } else {
      dst[e] = from_f32<OUT>((float)src[e] * s);
    }
  }
}

// Largest row width: a cluster of eight CTAs of 1024 threads with two groups of eight each.
constexpr int ROW_MAX = MAX_CLUSTER * 1024 * 2 * 8;

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

template <int KIND, bool VEC>
cudaError_t launch_shape(RowParams p, int n, cudaStream_t st) {
  const int groups = (p.k + 7) / 8;
  p.cluster = 1;
  if (groups <= 1024) return launch_pdl(row_int8_kernel<KIND, VEC, 1, false>, dim3(n), dim3((groups + 31) / 32 * 32), 0, st, p);
  if (groups <= 2048) return launch_pdl(row_int8_kernel<KIND, VEC, 2, false>, dim3(n), dim3((groups + 63) / 64 * 32), 0, st, p);
  while (p.cluster * 2048 < groups) p.cluster *= 2;
  const int t = (groups + 2 * p.cluster - 1) / (2 * p.cluster);
  return launch_pdl_cluster(row_int8_kernel<KIND, VEC, 2, true>, dim3(n * p.cluster), dim3((t + 31) / 32 * 32), p.cluster, 0, st, p);
}

// `esize`: bytes of one input element; the wide path wants whole groups of eight and 16-byte addresses on every row
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
  const cudaError_t e = vec ? launch_shape<KIND, true>(p, n, st) : launch_shape<KIND, false>(p, n, st);
  return (int)e;
}

template <typename OUT>
int launch_dequant(const signed char* q, long long ldq, const float* scale, void* out, long long ldo, int n, int k,
                   cudaStream_t st) {
  const bool vec = k % 8 == 0 && aligned(q, 8) && aligned(out, 16) && (n == 1 || (ldq % 8 == 0 && (ldo * sizeof(OUT)) % 16 == 0));
  const int per = 256 * (vec ? 8 : 1);
  const dim3 grid(n, min((k + per - 1) / per, 64));
  OUT* o = static_cast<OUT*>(out);
  return (int)(vec ? launch_pdl(dequant_int8_kernel<OUT, true>, grid, dim3(256), 0, st, q, ldq, scale, o, ldo, k)
                   : launch_pdl(dequant_int8_kernel<OUT, false>, grid, dim3(256), 0, st, q, ldq, scale, o, ldo, k));
}
}  // namespace

extern "C" int vg_quant_int8(const void* x, long long ldx, int dtype, int n, int k, void* q, long long ldq, float* scale,
                             cudaStream_t st) {
  RowParams p{};
  p.x = x; p.ldx = ldx; p.k = k; p.q = static_cast<signed char*>(q); p.ldq = ldq; p.scale = scale;
  switch (dtype) {
    case ROW_BF16: return launch_row<ROW_BF16>(p, n, 2, st);
    case ROW_F16: return launch_row<ROW_F16>(p, n, 2, st);
    case ROW_F32: return launch_row<ROW_F32>(p, n, 4, st);
  }
  return -2;
}

extern "C" int vg_swiglu_int8(const void* gu, long long ldx, int n, int inter, void* q, long long ldq, float* scale,
                              cudaStream_t st) {
  RowParams p{};
  p.x = gu; p.ldx = ldx; p.k = inter; p.q = static_cast<signed char*>(q); p.ldq = ldq; p.scale = scale;
  return launch_row<ROW_SWIGLU>(p, n, 2, st);
}

extern "C" int vg_add_rmsnorm_int8(void* res, long long ld_res, const void* delta, long long ld_delta, const float* w, int n,
                                   int h, float eps, int plus_one, void* q, long long ldq, float* scale, void* out16,
                                   long long ld_out16, cudaStream_t st) {
  RowParams p{};
  p.x = res; p.ldx = ld_res; p.delta = static_cast<const __nv_bfloat16*>(delta); p.ldd = ld_delta; p.w = w; p.k = h;
  p.eps = eps; p.w_off = plus_one ? 1.0f : 0.0f; p.q = static_cast<signed char*>(q); p.ldq = ldq; p.scale = scale;
  p.out16 = static_cast<__half*>(out16); p.ldo = ld_out16;
  return launch_row<ROW_NORM>(p, n, 2, st);
}

extern "C" int vg_dequant_int8(const void* q, long long ldq, const float* scale, void* out, long long ldo, int dtype, int n,
                               int k, cudaStream_t st) {
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
