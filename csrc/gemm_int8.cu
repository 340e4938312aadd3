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
    if (elect_one()) {
      pdl_wait();
      int st = 0;
      uint32_t ph = 1;
      for (int s = s0; s < s1; ++s) {
        if (!mbar_wait(empty + st, ph)) { fail(VG_ERR_EMPTY_WAIT); break; }
        uint8_t* a = smem + st * S::STAGE;
        mbar_arrive_expect_tx(full + st, S::STAGE);
        tma_tensor2d_g2s(a, &tm_w, s * BK, m0, full + st);
        tma_tensor2d_g2s(a + A_BYTES, &tm_x, s * BK, n0, full + st);
        if (++st == S::STAGES) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_i8(BM, BN);
    const uint64_t adesc0 = umma_desc_sw128(smem_u32(smem)), bdesc0 = umma_desc_sw128(smem_u32(smem) + A_BYTES);
    int st = 0;
    uint32_t ph = 0;
    for (int s = s0; s < s1; ++s) {
      if (!mbar_wait(full + st, ph)) { fail(VG_ERR_TMA_WAIT); break; }
      tc_fence_after();
      if (elect_one()) {
        const uint64_t off = (uint64_t)(st * (S::STAGE >> 4));
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk)
          umma_i8(tmem, adesc0 + off + kk * 2, bdesc0 + off + kk * 2, idesc, (s > s0 || kk) ? 1u : 0u);
        umma_commit(empty + st);
        if (s == s1 - 1) umma_commit(acc_full);
      }
      __syncwarp();
      if (++st == S::STAGES) { st = 0; ph ^= 1; }
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
  if (warp >= 2 && s1 > s0) {
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

// ------------------------------------------------------------------ wide form: CTA pairs
// Enough tokens to keep the tensor cores busy: a pair of CTAs (cta_group::2) owns 256 channels x BN tokens, each CTA
// loads its 128 channels and half of the tokens, so a byte of either operand that comes from L2 feeds twice the MMA work
// of a single-CTA tile (the 16 KB + BN * 64 B that a CTA fetches per slab is what bounds this kernel, not the MMAs).
// Persistent: one pair per two SMs walks the tiles with two accumulators in TMEM, so a tile's stores run under the next
// tile's MMAs. Tiles go token-first within groups of PAIR_GROUP token tiles: the weights of the running tiles and the
// group's tokens stay in L2.
constexpr int PBN = 256;                                  // token tile at most; BN is any multiple of 32 up to it
constexpr int P_STAGE = A_BYTES + PBN / 2 * BK;           // 32 KB
constexpr int P_STAGES = 6;
constexpr int P_SX = P_STAGES * P_STAGE;                  // [4 warps][PBN] token scales
constexpr int P_BARS = P_SX + 4 * PBN * 4;
constexpr int P_SMEM = P_BARS + 256 + 1024;
constexpr int PAIR_GROUP = 16;

VG_DEVINL void tma_pair_g2s(uint32_t dst, const void* tmap, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(dst), "l"(tmap), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
VG_DEVINL void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrives on the barrier at this offset in both CTAs of the pair once the MMAs issued so far are done
VG_DEVINL void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
VG_DEVINL void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
VG_DEVINL void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

struct PairTiles {
  int mt, nt, total;
  VG_DEVINL void at(int t, int& m, int& n) const {
    const int per = PAIR_GROUP * mt, g = t / per, first = g * PAIR_GROUP;
    const int width = min(PAIR_GROUP, nt - first), in = t - g * per;
    m = in / width;
    n = first + in % width;
  }
};

template <bool F32>
__global__ void __launch_bounds__(THREADS, 1)
gemm_int8_pair_kernel(const I8Params p, const int bn, const PairTiles tiles, const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_x) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + P_BARS);      // the leader's counts both CTAs' copies
  uint64_t* empty = full + P_STAGES;
  uint64_t* acc_full = empty + P_STAGES;                             // [2]
  uint64_t* acc_empty = acc_full + 2;                                // [2], the leader's counts both CTAs' epilogue warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int slabs = (p.K + BK - 1) / BK;
  pdl_trigger();

  if (threadIdx.x == 0) {
    for (int i = 0; i < P_STAGES; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                                // both CTAs' barriers are set up
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto fail = [&](int code) { if (p.err) atomicCAS(p.err, 0, code); *abort_flag = 1; };

  if (warp == 0) {
    if (elect_one()) {
      pdl_wait();
      const uint32_t tx = 2 * (uint32_t)(A_BYTES + bn / 2 * BK);
      const uint32_t full0 = dsmem_map(smem_u32(full), 0);
      int st = 0, issued = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (int t = pair; t < tiles.total && ok; t += npairs) {
        int mi, ni;
        tiles.at(t, mi, ni);
        const int m0 = mi * 2 * BM + rank * BM, n0 = ni * bn + rank * (bn / 2);
        for (int s = 0; s < slabs; ++s) {
          if (!mbar_wait(empty + st, ph)) { fail(VG_ERR_EMPTY_WAIT); ok = false; break; }
          const uint32_t a = smem_u32(smem + st * P_STAGE), bar = full0 + st * 8;
          if (rank == 0) mbar_arrive_expect_tx(full + st, tx);
          tma_pair_g2s(a, &tm_w, s * BK, m0, bar);
          tma_pair_g2s(a + A_BYTES, &tm_x, s * BK, n0, bar);
          ++issued;
          if (++st == P_STAGES) { st = 0; ph ^= 1; }
        }
      }
      // the pair's last commits have arrived here before this CTA may end
      for (int i = 0; i < min(issued, P_STAGES) && ok; ++i) {
        if (issued < P_STAGES) { st = i; ph = 0; }
        if (!mbar_wait(empty + st, ph)) { fail(VG_ERR_EMPTY_WAIT); ok = false; }
        if (issued >= P_STAGES && ++st == P_STAGES) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    // The whole warp walks the loop and one elected lane issues: descriptors then stay in uniform registers. (With the
    // loop inside a lane == 0 branch each MMA took 70 cycles to issue and a slab 330 more: 0.35 us a slab at any width.)
    if (rank == 0) {
      const uint32_t idesc = idesc_i8(2 * BM, bn);
      const uint64_t adesc0 = umma_desc_sw128(smem_u32(smem)), bdesc0 = umma_desc_sw128(smem_u32(smem) + A_BYTES);
      int st = 0, it = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = pair; t < tiles.total && ok; t += npairs, ++it) {
        const int buf = it & 1;
        if (!mbar_wait(acc_empty + buf, ((it >> 1) & 1) ^ 1)) { fail(VG_ERR_MMA_WAIT); break; }
        tc_fence_after();
        const uint32_t acc = tmem + buf * PBN;
        for (int s = 0; s < slabs; ++s) {
          if (!mbar_wait(full + st, ph)) { fail(VG_ERR_TMA_WAIT); ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t off = (uint64_t)(st * (P_STAGE >> 4));
#pragma unroll
            for (int kk = 0; kk < BK / 32; ++kk)
              umma_i8_pair(acc, adesc0 + off + kk * 2, bdesc0 + off + kk * 2, idesc, (s || kk) ? 1u : 0u);
            umma_commit_pair(empty + st);
            if (s == slabs - 1) umma_commit_pair(acc_full + buf);
          }
          __syncwarp();
          if (++st == P_STAGES) { st = 0; ph ^= 1; }
        }
      }
    }
  } else {
    pdl_wait();
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    float* sx = reinterpret_cast<float*>(smem + P_SX) + quarter * PBN;
    const uint32_t acc_empty0 = dsmem_map(smem_u32(acc_empty), 0);
    int it = 0;
    for (int t = pair; t < tiles.total; t += npairs, ++it) {
      const int buf = it & 1;
      int mi, ni;
      tiles.at(t, mi, ni);
      const int m = mi * 2 * BM + rank * BM + r, n0 = ni * bn;
      const int cols = min(bn, p.N - n0);
      __syncwarp();
      for (int c = lane; c < cols; c += 32) sx[c] = __ldg(p.sx + n0 + c);
      const float sw = m < p.M ? __ldg(p.sw + m) : 0.f;
      __syncwarp();
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full + buf, (it >> 1) & 1))) { fail(VG_ERR_MMA_WAIT); break; }
      tc_fence_after();
      const uint32_t acc = tmem + buf * PBN + ((uint32_t)(quarter * 32) << 16);
      for (int c = 0; c < cols; c += 32) {
        uint32_t v[32];
        tmem_ld32(acc + c, v);
        tmem_ld_wait();
        if (m < p.M) {
          char* o = static_cast<char*>(p.out) + ((size_t)(n0 + c) * p.ldo + m) * (F32 ? 4 : 2);
          const size_t step = (size_t)p.ldo * (F32 ? 4 : 2);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (c + i < cols) {
              const float y = (float)(int)v[i] * sw * sx[c + i];
              if (F32) *reinterpret_cast<float*>(o + i * step) = y;
              else *reinterpret_cast<__nv_bfloat16*>(o + i * step) = __float2bfloat16_rn(y);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty0 + buf * 8);
    }
  }
  __syncwarp();
  if (*abort_flag && threadIdx.x == 0) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);       // let copies in flight land before the block ends
  }
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
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

int sm_count(int dev) {
  static std::atomic<int> known[64];
  int n = known[dev & 63].load();
  if (n <= 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    known[dev & 63].store(n);
  }
  return n;
}

// The attribute belongs to the device's copy of a kernel: set once per kernel and device.
int allow_smem(const void* kernel, int bytes, int dev, std::atomic<unsigned long long>& done) {
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load() & bit) return 0;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit);
  return (int)e;
}

template <bool F32>
int launch_pair(const I8Params& p, int bn, int pairs, int dev, const CUtensorMap& tw, const CUtensorMap& tx, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  const int rc = allow_smem(reinterpret_cast<const void*>(gemm_int8_pair_kernel<F32>), P_SMEM, dev, done);
  if (rc) return rc;
  PairTiles t;
  t.mt = (p.M + 2 * BM - 1) / (2 * BM);
  t.nt = (p.N + bn - 1) / bn;
  t.total = t.mt * t.nt;
  return (int)launch_pdl_cluster(gemm_int8_pair_kernel<F32>, dim3(2 * min(pairs, t.total)), dim3(THREADS), 2u, P_SMEM, st, p, bn, t,
                                 tw, tx);
}

template <int BN>
int launch(const I8Params& p, int dev, const CUtensorMap& tw, const CUtensorMap& tx, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  const int rc = allow_smem(reinterpret_cast<const void*>(gemm_int8_kernel<BN>), Shape<BN>::SMEM, dev, done);
  if (rc) return rc;
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
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  const int sms = sm_count(dev);
  if (sms <= 0) return -3;
  const int bn = N <= 16 ? 16 : N <= 32 ? 32 : N <= 64 ? 64 : N <= 128 ? 128 : 256;
  const int tiles = (M + BM - 1) / BM, ntile = (N + bn - 1) / bn, slabs = (K + BK - 1) / BK;
  if (ntile > 65535 || (long long)tiles * ntile > (1 << 28)) return -2;
  I8Params p{};
  p.sx = sx; p.sw = sw; p.out = out; p.ldo = ldo; p.M = M; p.N = N; p.K = K; p.out_f32 = out_f32; p.err = err;
  // one CTA per SM at most while K is split, and at least four slabs per CTA
  p.split = max(1, min(MAX_SPLIT, min(sms / (tiles * ntile), slabs / 4)));
  CUtensorMap tw, tx;
  int rc = make_map(codes, M, K, ldw, BM, &tw);
  if (rc) return rc;
  if (N > 256) {
    const int nt = (N + PBN - 1) / PBN, pbn = ((N + nt - 1) / nt + 31) / 32 * 32;
    rc = make_map(q, N, K, ldq, pbn / 2, &tx);
    if (rc) return rc;
    return out_f32 ? launch_pair<true>(p, pbn, sms / 2, dev, tw, tx, st) : launch_pair<false>(p, pbn, sms / 2, dev, tw, tx, st);
  }
  rc = make_map(q, N, K, ldq, bn, &tx);
  if (rc) return rc;
  switch (bn) {
    case 16: return launch<16>(p, dev, tw, tx, st);
    case 32: return launch<32>(p, dev, tw, tx, st);
    case 64: return launch<64>(p, dev, tw, tx, st);
    case 128: return launch<128>(p, dev, tw, tx, st);
    default: return launch<256>(p, dev, tw, tx, st);
  }
}
