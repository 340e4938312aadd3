// Integer matrix product of the W8A8 path on the 5th-generation tensor cores (tcgen05.mma kind::i8).
//
//   out[n, m] = (sum_k q[n, k] * c[m, k]) * sx[n] * sw[m]
//
// q: int8 tokens with a scale each, c: int8 weights with a scale per output channel, both row-major as the quantisers
// write them. The sum is exact: int32 accumulators cannot overflow for K <= 131071 (128 * 128 * K < 2^31), so neither
// the tile shape nor the split of K shows in the result and a token's bits do not depend on the batch.
//
// Weights are the A operand (128 output channels = the 128 TMEM lanes), BN tokens the B operand. Slabs of 128 bytes of
// K of both arrive by tiled TMA with the 128-byte swizzle (zeros beyond K, the channels and the tokens).
// CTA (192 threads): warp 0 copies, warp 1 issues four K = 32 MMAs per slab, warps 2-5 read the accumulator back,
// thread = output channel, so a warp stores 32 neighbouring channels of one token. With few tiles K is split over a
// cluster: every CTA sends the columns of its partial sums to the CTA that owns them (distributed shared memory).
// All waits are bounded.
#include <cuda.h>
#include <atomic>
#include <mutex>

#include "common.cuh"
#include "api.h"

namespace {
using namespace vg;

constexpr int BM = 128;
constexpr int BK = 128;                     // bytes of K per slab
constexpr int A_BYTES = BM * BK;
constexpr int THREADS = 192;
constexpr int MAX_SPLIT = 8;

struct I8Params {
  const float* sx;
  const float* sw;
  void* out;
  long long ldo;
  int M, N, K, split, out_f32;
  int* err;
};

// Instruction descriptor: int32 accumulator, signed int8 operands, both K-major.
constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
VG_DEVINL void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
VG_DEVINL void dsmem_st_s32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

template <int BN>
struct Shape {
  static constexpr int B_BYTES = BN * BK;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  // two CTAs per SM while the token tile is small (the weight stream wants many loads in flight), else one
  static constexpr int CTAS = BN <= 64 ? 2 : 1;
  static constexpr int STAGES = (CTAS == 2 ? 108 : 216) * 1024 / STAGE;
  static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  static constexpr int SMEM = STAGES * STAGE + 1024 + 256;
  static_assert(STAGES * 16 + 32 <= 256, "barrier area");
};

// `v` holds columns [c0, c0 + 8) of this thread's channel.
VG_DEVINL void store8(const I8Params& p, int m, int n0, const uint32_t* v, float sw) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + i;
    if (n < p.N) {
      const float y = (float)(int)v[i] * sw * __ldg(p.sx + n);
      if (p.out_f32) static_cast<float*>(p.out)[(size_t)n * p.ldo + m] = y;
      else static_cast<__nv_bfloat16*>(p.out)[(size_t)n * p.ldo + m] = __float2bfloat16_rn(y);
    }
  }
}

template <int BN>
__global__ void __launch_bounds__(THREADS, Shape<BN>::CTAS)
gemm_int8_kernel(const I8Params p, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x) {
  using S = Shape<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::STAGES * S::STAGE);
  uint64_t* empty = full + S::STAGES;
  uint64_t* acc_full = empty + S::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.split > 1 ? (int)cluster_ctarank() : 0;
  const int m0 = (blockIdx.x / p.split) * BM, n0 = blockIdx.y * BN;
  const int slabs = (p.K + BK - 1) / BK;
  const int s0 = (int)((long long)slabs * rank / p.split), s1 = (int)((long long)slabs * (rank + 1) / p.split);
  pdl_trigger();

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto fail = [&](int code) { if (p.err) atomicCAS(p.err, 0, code); *abort_flag = 1; };

  if (warp == 0) {
    if (lane == 0) {
      pdl_wait();
      int st = 0;
      uint32_t ph = 1;
      for (int s = s0; s < s1 && !*abort_flag; ++s) {
        if (!mbar_wait(empty + st, ph)) { fail(VG_ERR_EMPTY_WAIT); break; }
        uint8_t* a = smem + st * S::STAGE;
        mbar_arrive_expect_tx(full + st, S::STAGE);
        tma_tensor2d_g2s(a, &tm_w, s * BK, m0, full + st);
        tma_tensor2d_g2s(a + A_BYTES, &tm_x, s * BK, n0, full + st);
        if (++st == S::STAGES) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8(BM, BN);
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int s = s0; s < s1 && !*abort_flag; ++s) {
        if (!mbar_wait(full + st, ph)) { fail(VG_ERR_TMA_WAIT); ok = false; break; }
        tc_fence_after();
        const uint32_t a = smem_u32(smem + st * S::STAGE), b = a + A_BYTES;
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk)
          umma_i8(tmem, umma_desc_sw128(a + kk * 32), umma_desc_sw128(b + kk * 32), idesc, (s > s0 || kk) ? 1u : 0u);
        umma_commit(empty + st);
        if (++st == S::STAGES) { st = 0; ph ^= 1; }
      }
      if (ok && s1 > s0) umma_commit(acc_full);
    }
  } else {
    pdl_wait();
  }
  __syncwarp();

  const int quarter = warp & 3;
  const int r = quarter * 32 + lane;                       // channel row of this thread within the tile
  const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
  const int cols = min(BN, p.N - n0);                      // columns that hold a token
  bool have = false;
  if (warp >= 2 && s1 > s0 && __all_sync(0xffffffffu, !*abort_flag)) {
    have = __all_sync(0xffffffffu, mbar_wait(acc_full, 0));
    if (!have) fail(VG_ERR_MMA_WAIT);
    tc_fence_after();
  }
  if (p.split == 1) {
    if (have) {
      const int m = m0 + r;
      const float sw = m < p.M ? p.sw[m] : 0.f;
      for (int c = 0; c < cols; c += 8) {
        uint32_t v[8];
        tmem_ld8(lane_base + c, v);
        tmem_ld_wait();
        if (m < p.M) store8(p, m, n0 + c, v, sw);
      }
    }
  } else {
    // columns [rank * own, ...) of the tile belong to cluster rank `rank`; its receive area (over the drained ring)
    // holds [source rank][column][channel]
    const int own = (BN + p.split - 1) / p.split;
    cluster_sync_all();                                    // every CTA's MMAs are done: the rings are free
    if (warp >= 2) {
      const uint32_t area = smem_u32(smem);
      for (int c = 0; c < cols; c += 8) {
        uint32_t v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (have) {
          tmem_ld8(lane_base + c, v);
          tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < cols)
            dsmem_st_s32(dsmem_map(area + (uint32_t)(((rank * own + (c + i) % own) * BM + r) * 4), (c + i) / own), v[i]);
      }
    }
    cluster_sync_all();
    if (warp >= 2) {
      const int m = m0 + r;
      const float sw = m < p.M ? p.sw[m] : 0.f;
      const int* area = reinterpret_cast<const int*>(smem);
      const int c1 = min(cols, (rank + 1) * own);
      for (int c = rank * own; c < c1; ++c) {
        int sum = 0;
        for (int q = 0; q < p.split; ++q) sum += area[(q * own + c - rank * own) * BM + r];
        if (m < p.M) {
          const float y = (float)sum * sw * __ldg(p.sx + n0 + c);
          if (p.out_f32) static_cast<float*>(p.out)[(size_t)(n0 + c) * p.ldo + m] = y;
          else static_cast<__nv_bfloat16*>(p.out)[(size_t)(n0 + c) * p.ldo + m] = __float2bfloat16_rn(y);
        }
      }
    }
  }
  if (*abort_flag && threadIdx.x == 0) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);       // let copies in flight land before the block ends
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, S::TMEM_COLS);
}

// ------------------------------------------------------------------ host
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn get_encode() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(f);
  });
  return fn;
}
// [rows][k] bytes with row pitch `ld`, box = one 128-byte slab x `box_rows`
int make_map(const void* base, int rows, int k, long long ld, int box_rows, CUtensorMap* out) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return -1;
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t str[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {BK, (cuuint32_t)box_rows}, one[2] = {1, 1};
  const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, str, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -(int)r - 100;
}

template <int BN>
int launch(const I8Params& p, const CUtensorMap& tw, const CUtensorMap& tx, cudaStream_t st) {
  // the attribute belongs to the device's copy of the kernel: set once per device
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(done.load() & bit)) {
    e = cudaFuncSetAttribute(gemm_int8_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<BN>::SMEM);
    if (e != cudaSuccess) return (int)e;
    done.fetch_or(bit);
  }
  const dim3 grid((unsigned)((p.M + BM - 1) / BM * p.split), (unsigned)((p.N + BN - 1) / BN));
  return (int)launch_pdl_cluster(gemm_int8_kernel<BN>, grid, dim3(THREADS), (unsigned)p.split, Shape<BN>::SMEM, st, p, tw, tx);
}
}  // namespace

extern "C" int vg_gemm_int8(const void* codes, long long ldw, const float* sw, const void* q, long long ldq, const float* sx,
                            void* out, long long ldo, int out_f32, int M, int K, int N, int* err, cudaStream_t st) {
  if (M <= 0 || N < 0 || K <= 0 || K > 131071 || ldw % 16 || ldq % 16 || ldw < K || ldq < K || ldo < M ||
      (reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(q)) % 16)
    return -2;
  if (N == 0) return 0;
  int sms = 0, dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return (int)e;
  const int bn = N <= 16 ? 16 : N <= 32 ? 32 : N <= 64 ? 64 : N <= 128 ? 128 : 256;
  const int tiles = (M + BM - 1) / BM, ntile = (N + bn - 1) / bn, slabs = (K + BK - 1) / BK;
  if (ntile > 65535) return -2;
  I8Params p{};
  p.sx = sx; p.sw = sw; p.out = out; p.ldo = ldo; p.M = M; p.N = N; p.K = K; p.out_f32 = out_f32; p.err = err;
  // one CTA per SM at most while K is split, and at least four slabs per CTA
  p.split = max(1, min(MAX_SPLIT, min(sms / (tiles * ntile), slabs / 4)));
  CUtensorMap tw, tx;
  int rc = make_map(codes, M, K, ldw, BM, &tw);
  if (rc) return rc;
  rc = make_map(q, N, K, ldq, bn, &tx);
  if (rc) return rc;
  switch (bn) {
    case 16: return launch<16>(p, tw, tx, st);
    case 32: return launch<32>(p, tw, tx, st);
    case 64: return launch<64>(p, tw, tx, st);
    case 128: return launch<128>(p, tw, tx, st);
    default: return launch<256>(p, tw, tx, st);
  }
}
