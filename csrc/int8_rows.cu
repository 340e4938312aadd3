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
#include <atomic>

#include "common.cuh"
#include "api.h"

namespace {
using namespace vg;

constexpr int MAX_CLUSTER = 8;
constexpr int RING_SLOTS = 8;
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
  int* err;
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

// Eight values -> eight codes, rint(v * f) for |v * f| < 2^22: adding 1.5 * 2^23 leaves the rounded integer in the low bits
// of the sum. (cvt.rni runs at an eighth of the rate, next to the exponentials.)
VG_DEVINL uint2 codes8(const float* v, float f) {
  uint32_t t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = __float_as_uint(__fmaf_rn(v[i], f, 12582912.0f));
  return make_uint2(__byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410));
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

// What a row's statistics give: the scale, its reciprocal and (norm) 1 / rms.
struct RowScale {
  float s, f, inv;
  bool bad;
};
template <int KIND>
VG_DEVINL RowScale row_scale(const RowParams& p, unsigned mx, float ss) {
  // The norm's factor 1 / rms is common to the row, so the maximum of |res * w| found in the same pass as the sum of
  // squares is enough: one reduction instead of two.
  RowScale o;
  o.inv = KIND == ROW_NORM ? rsqrtf(ss / (float)p.k + p.eps) : 1.f;
  const float amax = __uint_as_float(mx) * o.inv;
  o.bad = !(amax < INFINITY) || (KIND == ROW_NORM && !(ss < INFINITY));
  o.s = o.bad ? __uint_as_float(0x7fffffffu) : fmaxf(__fdiv_rn(amax, INT8_MAX_CODE), SCALE_FLOOR);
  // codes are rint(y * (1 / s)): |y| / s <= 127 (1 + 2^-22), which rounds to 127 at most; 1 / s <= 2^120
  o.f = o.bad ? 0.f : __fdiv_rn(1.f, o.s);
  return o;
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

  const RowScale rs = row_scale<KIND>(p, mx, ss);
  if (tid == 0) p.scale[row] = rs.s;
  if (KIND == ROW_NORM) {
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] *= rs.inv;
  }
  signed char* q = p.q + row * p.ldq;
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    if (VEC) {
      const int e = (tid + c * T) * 8;
      if (e < k) {
        *reinterpret_cast<uint2*>(q + e) = rs.bad ? make_uint2(0u, 0u) : codes8(v[c], rs.f);
        if (KIND == ROW_NORM && p.out16) {
          uint4 h4;
          __half* h = reinterpret_cast<__half*>(&h4);
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = rs.bad ? __ushort_as_half(0x7fff) : f32_to_f16_sat(v[c][i]);
          *reinterpret_cast<uint4*>(p.out16 + row * p.ldo + e) = h4;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = tid + (c * 8 + i) * T;
        if (e < k) {
          q[e] = (signed char)(rs.bad ? 0 : __float2int_rn(v[c][i] * rs.f));
          if (KIND == ROW_NORM && p.out16)
            p.out16[row * p.ldo + e] = rs.bad ? __ushort_as_half(0x7fff) : f32_to_f16_sat(v[c][i]);
        }
      }
    }
  }
}

// Many rows: persistent blocks with a ring of whole rows in shared memory, filled by bulk copies several rows ahead, so
// the memory system stays busy while a block reduces, quantises and stores. A row's slot is refilled as soon as the
// reduction's barrier has shown that every thread holds its part in registers: one barrier per row.
template <int KIND, int MAXC>
__global__ void __launch_bounds__(MAXC == 4 ? 640 : 1024) row_int8_ring_kernel(const RowParams p, int n, int slots, int slot_bytes) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[RING_SLOTS];
  __shared__ unsigned red_m[2][32];
  __shared__ float red_s[2][32];
  __shared__ int stuck;
  constexpr int ES = KIND == ROW_F32 ? 4 : 2;
  pdl_trigger();
  const int k = p.k, T = blockDim.x, step = gridDim.x;
  const uint32_t x_bytes = (uint32_t)k * ES * (KIND == ROW_SWIGLU ? 2 : 1);
  const bool two = KIND == ROW_NORM && p.delta;
  if (threadIdx.x == 0) {
    for (int i = 0; i < slots; ++i) mbar_init(full + i, 1);
    stuck = 0;
    fence_mbar_init();
  }
  __syncthreads();
  auto fill = [&](int slot, size_t row) {
    uint8_t* dst = ring + (size_t)slot * slot_bytes;
    mbar_arrive_expect_tx(full + slot, two ? 2 * x_bytes : x_bytes);
    tma_bulk_g2s(dst, static_cast<const char*>(p.x) + row * p.ldx * ES, x_bytes, full + slot);
    if (two) tma_bulk_g2s(dst + x_bytes, p.delta + row * p.ldd, x_bytes, full + slot);
  };
  pdl_wait();
  if (threadIdx.x == 0)
    for (int i = 0; i < slots && (int)blockIdx.x + i * step < n; ++i) fill(i, blockIdx.x + (size_t)i * step);
  int slot = 0, it = 0;
  uint32_t ph = 0;
  for (int row = blockIdx.x; row < n; row += step, ++it) {
    if (!mbar_wait(full + slot, ph)) {
      if (p.err) atomicCAS(p.err, 0, (int)VG_ERR_TMA_WAIT);
      stuck = 1;
    }
    const uint8_t* src = ring + (size_t)slot * slot_bytes;
    float v[MAXC][8];
    unsigned mx = 0;
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < MAXC; ++c) {
      const int e = (threadIdx.x + c * T) * 8;
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
          const float4 w0 = __ldg(reinterpret_cast<const float4*>(p.w + e)), w1 = __ldg(reinterpret_cast<const float4*>(p.w + e + 4));
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
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(v[c][i]) & 0x7fffffffu);
    }
    block_reduce<KIND == ROW_NORM>(mx, ss, red_m[it & 1], red_s[it & 1]);
    if (stuck) break;                                      // seen by every thread: set before the barrier
    if (threadIdx.x == 0 && row + (long long)slots * step < n) fill(slot, row + (size_t)slots * step);
    const RowScale rs = row_scale<KIND>(p, mx, ss);
    if (threadIdx.x == 0) p.scale[row] = rs.s;
#pragma unroll
    for (int c = 0; c < MAXC; ++c) {
      const int e = (threadIdx.x + c * T) * 8;
      if (e < k) {
        if (KIND == ROW_NORM) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] *= rs.inv;
        }
        *reinterpret_cast<uint2*>(p.q + (size_t)row * p.ldq + e) = rs.bad ? make_uint2(0u, 0u) : codes8(v[c], rs.f);
        if (KIND == ROW_NORM && p.out16) {
          const uint4 nan4 = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
          *reinterpret_cast<uint4*>(p.out16 + (size_t)row * p.ldo + e) = rs.bad ? nan4 : pack_f16_sat(v[c]);
        }
      }
    }
    if (++slot == slots) { slot = 0; ph ^= 1; }
  }
  if (stuck && threadIdx.x == 0)
    for (int i = 0; i < 64; ++i) __nanosleep(1000);        // let copies in flight land before the block ends
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

constexpr int RING_BYTES = 200 * 1024;            // ring of all blocks of an SM
constexpr int RING_PER_SM = 4;                    // blocks per SM
constexpr int RING_MIN_ROWS = 2;                  // rows per SM from which the ring form pays

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

int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  n = known[dev & 63].load();
  if (n <= 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) known[dev & 63].store(n);
  return n;
}

template <int KIND, int MAXC>
int launch_ring(const RowParams& p, int n, int slot_bytes, int sms, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (!(done.load() & (1ull << (dev & 63)))) {
    e = cudaFuncSetAttribute(row_int8_ring_kernel<KIND, MAXC>, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES);
    if (e != cudaSuccess) return (int)e;
    done.fetch_or(1ull << (dev & 63));
  }
  const int groups = p.k / 8, threads = ((groups + MAXC - 1) / MAXC + 31) / 32 * 32;
  const int per_sm = max(1, min(min(RING_PER_SM, 1536 / threads), RING_BYTES / (2 * slot_bytes)));
  const int slots = max(2, min(RING_SLOTS, RING_BYTES / per_sm / slot_bytes));
  const int grid = min(n, sms * per_sm);
  return (int)launch_pdl(row_int8_ring_kernel<KIND, MAXC>, dim3(grid), dim3(threads), (size_t)slots * slot_bytes, st, p, n, slots, slot_bytes);
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
  const int sms = sm_count(), slot = p.k * esize * ((KIND == ROW_SWIGLU || p.delta) ? 2 : 1);
  if (vec && n >= RING_MIN_ROWS * sms && slot % 16 == 0 && 2 * slot <= RING_BYTES && p.k <= 640 * 32) {
    const int groups = p.k / 8;
    return groups <= 32 ? launch_ring<KIND, 1>(p, n, slot, sms, st)
           : groups <= 1024 ? launch_ring<KIND, 2>(p, n, slot, sms, st)
                            : launch_ring<KIND, 4>(p, n, slot, sms, st);
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
  p.eps = eps; p.w_off = plus_one ? 1.0f : 0.0f; p.q = static_cast<signed char*>(q); p.ldq = ldq; p.scale = scale; p.err = err;
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
