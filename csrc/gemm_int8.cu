// Integer matrix product of the W8A8 path on the 5th-generation tensor cores (tcgen05.mma kind::i8).
//
//   out[n, m] = (sum_k q[n, k] * c[m, k]) * sw[m] * sx[n]
//
// q: int8 tokens with a scale each, c: int8 weights with a scale per output channel, both row-major as the quantisers
// write them. The sum is exact: int32 accumulators cannot overflow for K <= 131071 (128 * 128 * K < 2^31), so neither
// the tile shape nor the split of K shows in the result and a token's bits do not depend on the batch.
//
// Weights are the A operand (output channels = the 128 TMEM lanes of a CTA), tokens the B operand. Slabs of 128 bytes of
// K of both arrive by tiled TMA with the 128-byte swizzle (zeros beyond K, the channels and the tokens). Two forms:
//   narrow  up to 64 tokens: one CTA per 128 channels, bound by the weight stream
//   pair    more: a pair of CTAs per 256 channels x up to 256 tokens (cta_group::2), bound by the MMAs
// In both warp 0 copies, warp 1 issues four K = 32 MMAs per slab, and four or eight more warps read the accumulator back,
// lane = output channel. With few tiles K is split over a cluster and the partial sums meet in distributed shared
// memory. All waits are bounded.
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
constexpr int NARROW_MAX = 64;              // tokens of the narrow form
constexpr int SX_PAD = 4;                   // read past a tile's last token scale, never used

struct I8Params {
  const float* sx;
  const float* sw;
  void* out;
  long long ldo;
  int M, N, K, split, out_f32;
  int vec;                                  // four channels of a token can be stored at once
  int* err;
};

// A value that is the same in all lanes, in a form the compiler knows to be: branches on it and descriptors made from it
// stay in uniform registers, which the MMA instructions need.
template <typename T>
VG_DEVINL T uniform(T v) { return (T)__shfl_sync(0xffffffffu, v, 0); }

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
VG_DEVINL void dsmem_st_v4(uint32_t addr, const uint32_t* v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// L2 only: safe before the wait for the predecessor kernel, which may still be writing these bytes (L2 is where its
// stores and the later loads meet)
VG_DEVINL void tma_prefetch_l2(const void* tmap, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(tmap), "r"(c0), "r"(c1) : "memory");
}
// Where a warp's stores go: 32 channels (this lane's is `m`) of the tokens from n0 on.
struct OutWarp {
  char* base;               // vec: token (lane & 3), the first of the four channels around this lane; else token 0, channel m
  size_t pitch;             // bytes between tokens
  float sw;
  bool in;                  // this lane has something to store
  VG_DEVINL OutWarp(const I8Params& p, int m, int n0) {
    const int lane = threadIdx.x & 31, es = p.out_f32 ? 4 : 2;
    pitch = (size_t)p.ldo * es;
    sw = m < p.M ? p.sw[m] : 0.f;
    in = m < p.M;           // vec needs M % 4 == 0: the four channels are inside or outside together
    base = static_cast<char*>(p.out) + (p.vec ? (size_t)(n0 + (lane & 3)) * pitch + (size_t)(m & ~3) * es
                                              : (size_t)n0 * pitch + (size_t)m * es);
  }
};

// Stores G groups of four columns (`v`, int32 sums of this lane's channel). Group g is columns c[g] .. c[g] + 3, of which
// those below `cols` hold a token; `sx` has the tile's token scales.
// A warp has 32 channels of one token per register, so storing registers as they are takes one 2-byte store per value and
// lane. The vec form transposes 4 x 4 blocks among neighbouring lanes first (two or four shuffles), then each lane stores
// four channels of one token. A scheduler has one or two of these warps, so what counts is that all groups' chains are
// independent and in one basic block: with a branch per group a 256-column tile took 11.4 k cycles, this way 5.4 k.
template <bool F32, bool VEC, int G>
VG_DEVINL void store_groups(const OutWarp& o, const int* c, int cols, const uint32_t* v, const float* sx) {
  const int lane = threadIdx.x & 31;
  const bool b0 = lane & 1, b1 = lane & 2;
  float y[G][4];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float4 s = *reinterpret_cast<const float4*>(sx + c[g]);
    y[g][0] = (float)(int)v[4 * g] * o.sw * s.x;
    y[g][1] = (float)(int)v[4 * g + 1] * o.sw * s.y;
    y[g][2] = (float)(int)v[4 * g + 2] * o.sw * s.z;
    y[g][3] = (float)(int)v[4 * g + 3] * o.sw * s.w;
  }
  if (!VEC) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        char* d = o.base + (size_t)(c[g] + i) * o.pitch;
        if (o.in && c[g] + i < cols) {
          if (F32) *reinterpret_cast<float*>(d) = y[g][i];
          else *reinterpret_cast<__nv_bfloat16*>(d) = __float2bfloat16_rn(y[g][i]);
        }
      }
    return;
  }
  if (F32) {
    float2 A[G], B[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float ra = __shfl_xor_sync(0xffffffffu, b0 ? y[g][0] : y[g][1], 1), rb = __shfl_xor_sync(0xffffffffu, b0 ? y[g][2] : y[g][3], 1);
      A[g] = b0 ? make_float2(ra, y[g][1]) : make_float2(y[g][0], ra);      // token b0, channels (even, odd)
      B[g] = b0 ? make_float2(rb, y[g][3]) : make_float2(y[g][2], rb);      // token 2 + b0
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float2 snd = b1 ? A[g] : B[g], own = b1 ? B[g] : A[g];
      const float2 rcv = make_float2(__shfl_xor_sync(0xffffffffu, snd.x, 2), __shfl_xor_sync(0xffffffffu, snd.y, 2));
      const float4 w = b1 ? make_float4(rcv.x, rcv.y, own.x, own.y) : make_float4(own.x, own.y, rcv.x, rcv.y);
      if (o.in && c[g] + (lane & 3) < cols) *reinterpret_cast<float4*>(o.base + (size_t)c[g] * o.pitch) = w;
    }
  } else {
    uint32_t w0[G], w1[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const __nv_bfloat162 e2 = __floats2bfloat162_rn(y[g][0], y[g][2]), o2 = __floats2bfloat162_rn(y[g][1], y[g][3]);
      const uint32_t e = *reinterpret_cast<const uint32_t*>(&e2), q = *reinterpret_cast<const uint32_t*>(&o2);
      const uint32_t own = b0 ? q : e, rcv = __shfl_xor_sync(0xffffffffu, b0 ? e : q, 1);
      const uint32_t lo = b0 ? rcv : own, hi = b0 ? own : rcv;              // even channel, odd channel
      w0[g] = __byte_perm(lo, hi, 0x5410);                                  // tokens b0 and 2 + b0
      w1[g] = __byte_perm(lo, hi, 0x7632);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t mine = b1 ? w1[g] : w0[g], other = __shfl_xor_sync(0xffffffffu, b1 ? w0[g] : w1[g], 2);
      const uint2 w = b1 ? make_uint2(other, mine) : make_uint2(mine, other);
      if (o.in && c[g] + (lane & 3) < cols) *reinterpret_cast<uint2*>(o.base + (size_t)c[g] * o.pitch) = w;
    }
  }
}
template <int G>
VG_DEVINL void store_columns(const I8Params& p, const OutWarp& o, const int* c, int cols, const uint32_t* v, const float* sx) {
  if (p.vec) {
    if (p.out_f32) store_groups<true, true, G>(o, c, cols, v, sx);
    else store_groups<false, true, G>(o, c, cols, v, sx);
  } else {
    if (p.out_f32) store_groups<true, false, G>(o, c, cols, v, sx);
    else store_groups<false, false, G>(o, c, cols, v, sx);
  }
}
// Accumulator columns [0, cols) of a whole tile, 4 * G at a time; `of` warps with the same channels take turns.
template <int G>
VG_DEVINL void store_tile(const I8Params& p, const OutWarp& o, uint32_t acc, int cols, const float* sx, int turn, int of) {
  for (int c0 = turn * 4 * G; c0 < cols; c0 += of * 4 * G) {
    uint32_t v[4 * G];
#pragma unroll
    for (int i = 0; i < G / 2; ++i) tmem_ld8(acc + c0 + 8 * i, v + 8 * i);
    tmem_ld_wait();
    int c[G];
#pragma unroll
    for (int g = 0; g < G; ++g) c[g] = c0 + 4 * g;
    store_columns<G>(p, o, c, cols, v, sx);
  }
}
// A warp's own copy of the token scales, fetched while the accumulator is still being built.
VG_DEVINL void fetch_sx(const I8Params& p, float* sx, int n0, int cols) {
  __syncwarp();
  for (int c = threadIdx.x & 31; c < (cols + 31) / 32 * 32; c += 32) sx[c] = c < cols ? p.sx[n0 + c] : 0.f;
  __syncwarp();
}

// Split K: columns go in groups of four, group g to the part g % parts. A part's receive area (over the drained ring)
// holds [source part][own group][channel] as 16-byte words. 64 x 5120 x 17408 in seven parts: sending takes 1.9 us and
// joining 1.7 of 19.0; 256 tokens in three parts 2.9 and 3.4 of 26.7. Sending moves 15 bytes a cycle and SM between SMs
// whatever the order of the parts, the columns read at a time (16, 32, 64) or the way the own part is kept.
VG_DEVINL uint32_t group_slots(int cols, int parts) { return (uint32_t)(((cols + 3) / 4 + parts - 1) / parts); }
// `to_rank(part)`: cluster rank of the CTA of that part which holds the same channels
template <typename F>
VG_DEVINL void send_partials(uint32_t area, uint32_t acc, int cols, int part, int parts, int r, int turn, int of, F to_rank) {
  const uint32_t slots = group_slots(cols, parts);
  for (int c = turn * 16; c < cols; c += of * 16) {
    uint32_t v[16] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    tmem_ld8(acc + c, v);
    if (c + 8 < cols) tmem_ld8(acc + c + 8, v + 8);
    tmem_ld_wait();
    uint32_t slot = (uint32_t)(c / 4) / (uint32_t)parts;
    int dst = c / 4 - (int)slot * parts;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c + 4 * i < cols) dsmem_st_v4(dsmem_map(area + ((part * slots + slot) * BM + r) * 16, to_rank(dst)), v + 4 * i);
      if (++dst == parts) { dst = 0; ++slot; }
    }
  }
}
// A part whose accumulator never came tells every part, itself among them: none stores a sum that lacks a piece of K.
template <typename F>
VG_DEVINL void report_lost(const volatile int* lost, int parts, F to_rank) {
  const int lane = threadIdx.x & 31;
  if (lane < parts) dsmem_st_u32(dsmem_map(smem_u32(const_cast<const int*>(lost)), to_rank(lane)), 1u);
}
template <int G>
VG_DEVINL void finish_partials(const I8Params& p, const uint8_t* area, const OutWarp& o, const float* sx, int cols, int part, int parts,
                               int r, int turn, int of) {
  const int slots = (int)group_slots(cols, parts);
  const uint4* a = reinterpret_cast<const uint4*>(area) + r;
  for (int s0 = turn * G; s0 < slots && (s0 * parts + part) * 4 < cols; s0 += of * G) {
    uint32_t v[4 * G] = {};
    int c[G];
    const uint4* at[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      // groups past the end come out as columns from the first multiple of four after `cols` on, which are not stored
      c[g] = min(((s0 + g) * parts + part) * 4, (cols + 3) / 4 * 4);
      at[g] = a + min(s0 + g, slots - 1) * BM;
    }
    for (int q = 0; q < parts; ++q)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint4 w = at[g][q * slots * BM];
        v[4 * g] += w.x; v[4 * g + 1] += w.y; v[4 * g + 2] += w.z; v[4 * g + 3] += w.w;
      }
    store_columns<G>(p, o, c, cols, v, sx);
  }
}

// ------------------------------------------------------------------ narrow form
template <int BN>
struct Shape {
  static constexpr int B_BYTES = BN * BK;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 108 * 1024 / STAGE;       // two CTAs per SM: the weight stream wants many loads in flight
  static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  static constexpr int SX = STAGES * STAGE + 256;         // [4 warps][NARROW_MAX + SX_PAD] token scales
  static constexpr int SMEM = SX + 4 * (NARROW_MAX + SX_PAD) * 4 + 1024;
  static_assert(STAGES * 16 + 32 <= 256, "barrier area");
  static_assert((BN / 4 + MAX_SPLIT) * BM * 16 <= STAGES * STAGE, "partial sums over the ring");
};

template <int BN>
__global__ void __launch_bounds__(THREADS, 2)
gemm_int8_kernel(const I8Params p, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x) {
  using S = Shape<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::STAGES * S::STAGE);
  uint64_t* empty = full + S::STAGES;
  uint64_t* acc_full = empty + S::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* lost = abort_flag + 1;                   // split: some part of this tile has no sums to send

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = p.split > 1 ? uniform((int)cluster_ctarank()) : 0;
  const int m0 = (blockIdx.x / p.split) * BM, n0 = blockIdx.y * BN;
  const int slabs = (p.K + BK - 1) / BK;
  const int s0 = (int)((long long)slabs * rank / p.split), s1 = (int)((long long)slabs * (rank + 1) / p.split);

  if (warp == 0 && elect_one()) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    for (int s = s0; s < min(s1, s0 + S::STAGES); ++s) tma_prefetch_l2(&tm_w, s * BK, m0);
  }
  if (threadIdx.x == 64) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    *lost = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Not before the allocation: a dependent that takes all 512 columns first would wait for this grid, and this grid for it.
  pdl_trigger();
  const uint32_t tmem = uniform(*tmem_slot);
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
    pdl_wait();                                           // no stage fills before: the bounded waits time this kernel's work only
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
  float* sx = reinterpret_cast<float*>(smem + S::SX) + quarter * (NARROW_MAX + SX_PAD);
  bool have = false;
  if (warp >= 2) {
    fetch_sx(p, sx, n0, cols);
    have = __all_sync(0xffffffffu, mbar_wait(acc_full, 0));
    if (!have) fail(VG_ERR_MMA_WAIT);
    tc_fence_after();
  }
  if (p.split == 1) {
    if (have) {
      store_tile<4>(p, OutWarp(p, m0 + r, n0), lane_base, cols, sx, 0, 1);
    }
  } else {
    cluster_sync_all();                                    // every CTA's MMAs are done: the rings are free
    auto to_rank = [](int q) { return (uint32_t)q; };
    if (warp >= 2) {
      if (have) send_partials(smem_u32(smem), lane_base, cols, rank, p.split, r, 0, 1, to_rank);
      else report_lost(lost, p.split, to_rank);
    }
    cluster_sync_all();
    if (warp >= 2 && !*lost) finish_partials<2>(p, smem, OutWarp(p, m0 + r, n0), sx, cols, rank, p.split, r, 0, 1);
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);       // let copies and MMAs in flight end before the block does
  }
  if (warp == 1) tmem_dealloc(tmem, S::TMEM_COLS);
}

// ------------------------------------------------------------------ pair form
// A pair of CTAs owns 256 channels x BN tokens; each loads its 128 channels and half of the tokens, so a byte of either
// operand that comes from L2 feeds twice the MMA work of a single-CTA tile. A slab takes 2 cycles per token of the tile
// (512 cycles at 256: the nominal rate of the tensor cores, seen with clock stamps), and copies keep up from 128 tokens on.
// Whole K: persistent, one pair per two SMs walks the tiles with two accumulators in TMEM, so a tile's stores run under
// the next tile's MMAs. Tiles go token-first within groups of PAIR_GROUP token tiles: the weights of the running tiles and
// the group's tokens stay in L2.
// Split K: a cluster of `split` pairs per tile, one tile per cluster.
constexpr int PBN = 256;                                  // token tile at most; BN is any multiple of 32 up to it
constexpr int P_RING = 216 * 1024;                        // stages of one or two slabs, 16 KB + 64 * BN bytes each
constexpr int P_MAX_STAGES = 8;
constexpr int P_EPI = 8;                                  // epilogue warps, two for each quarter of the channels
constexpr int P_THREADS = 64 + 32 * P_EPI;
constexpr int P_SX = P_RING;                              // [P_EPI warps][PBN + SX_PAD] token scales
constexpr int P_BARS = P_SX + P_EPI * (PBN + SX_PAD) * 4;
constexpr int P_SMEM = P_BARS + 256 + 1024;
constexpr int PAIR_GROUP = 16;
constexpr int PAIR_MAX_SPLIT = 4;
static_assert((PBN / 4 + PAIR_MAX_SPLIT) * BM * 16 <= P_RING, "partial sums over the ring");
static_assert(P_MAX_STAGES * 16 + 48 <= 256, "barrier area");

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
VG_DEVINL void umma_commit_pair(uint64_t* bar, uint16_t pair_mask) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"(pair_mask)
      : "memory");
}
VG_DEVINL void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
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

struct PairShape {
  int bn, b_slab, per, stage, stages;                    // token tile, bytes of a CTA's token slab, slabs and bytes of a stage, stages
  PairTiles tiles;
};

template <bool SPLIT>
__global__ void __launch_bounds__(P_THREADS, 1)
gemm_int8_pair_kernel(const I8Params p, const PairShape sh, const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_x) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + P_BARS);      // the leader's counts both CTAs' copies
  uint64_t* empty = full + P_MAX_STAGES;
  uint64_t* acc_full = empty + P_MAX_STAGES;                         // [2]
  uint64_t* acc_empty = acc_full + 2;                                // [2], the leader's counts both CTAs' epilogue warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* lost = abort_flag + 1;                   // split: some part of this tile has no sums to send

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int crank = uniform((int)cluster_ctarank());
  const int rank = crank & 1, leader = crank & ~1;                   // within the pair / the pair's first CTA
  const int part = SPLIT ? crank >> 1 : 0;
  const int first = SPLIT ? (int)blockIdx.x / (2 * p.split) : (int)blockIdx.x >> 1;
  const int step = SPLIT ? sh.tiles.total : (int)gridDim.x >> 1;     // split: one tile per cluster
  const int slabs = (p.K + BK - 1) / BK;
  const int s0 = SPLIT ? (int)((long long)slabs * part / p.split) : 0;
  const int s1 = SPLIT ? (int)((long long)slabs * (part + 1) / p.split) : slabs;

  if (warp == 0 && elect_one()) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    int mi, ni;
    sh.tiles.at(first, mi, ni);
    for (int s = s0; s < min(s1, s0 + sh.per * sh.stages); ++s) tma_prefetch_l2(&tm_w, s * BK, mi * 2 * BM + rank * BM);
  }
  if (threadIdx.x == 64) {
    for (int i = 0; i < sh.stages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, 2 * P_EPI);
    }
    *abort_flag = 0;
    *lost = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                                // both CTAs' barriers are set up
  tc_fence_after();
  pdl_trigger();                                                     // not before the allocation, as above
  const uint32_t tmem = uniform(*tmem_slot);
  // both CTAs of the pair have to know: copies of either signal the leader, MMAs read both
  auto fail = [&](int code) {
    if (p.err) atomicCAS(p.err, 0, code);
    *abort_flag = 1;
    dsmem_st_u32(dsmem_map(smem_u32(const_cast<const int*>(abort_flag)), crank ^ 1), 1u);
  };

  const int quarter = warp & 3;
  const int r = quarter * 32 + lane;                                 // channel of this thread within the CTA's 128
  const int turn = (warp - 2) >> 2;                                  // which of the quarter's two epilogue warps
  float* sx = reinterpret_cast<float*>(smem + P_SX) + (warp - 2) * (PBN + SX_PAD);
  bool have = false;
  if (warp == 0) {
    if (elect_one()) {
      int mi, ni;
      pdl_wait();
      const uint32_t full0 = dsmem_map(smem_u32(full), leader);
      int st = 0, issued = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (int t = first; t < sh.tiles.total && ok; t += step) {
        sh.tiles.at(t, mi, ni);
        const int m0 = mi * 2 * BM + rank * BM, n0 = ni * sh.bn + rank * (sh.bn / 2);
        for (int s = s0; s < s1; s += sh.per) {
          if (!mbar_wait(empty + st, ph)) { fail(VG_ERR_EMPTY_WAIT); ok = false; break; }
          const uint32_t a = smem_u32(smem) + st * sh.stage, b = a + sh.per * A_BYTES, bar = full0 + st * 8;
          const bool both = sh.per == 2 && s + 1 < s1;
          if (rank == 0) mbar_arrive_expect_tx(full + st, (both ? 4 : 2) * (uint32_t)(A_BYTES + sh.b_slab));
          tma_pair_g2s(a, &tm_w, s * BK, m0, bar);
          tma_pair_g2s(b, &tm_x, s * BK, n0, bar);
          if (both) {
            tma_pair_g2s(a + A_BYTES, &tm_w, s * BK + BK, m0, bar);
            tma_pair_g2s(b + sh.b_slab, &tm_x, s * BK + BK, n0, bar);
          }
          ++issued;
          if (++st == sh.stages) { st = 0; ph ^= 1; }
        }
      }
      // the pair's last commits have arrived here before this CTA may end
      if (issued < sh.stages) { st = 0; ph = 0; }
      for (int i = 0; i < min(issued, sh.stages) && ok; ++i) {
        if (!mbar_wait(empty + st, ph)) { fail(VG_ERR_EMPTY_WAIT); ok = false; }
        if (++st == sh.stages) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    // The whole warp walks the loop and one elected lane issues. A stage costs 260 cycles of waiting, electing and
    // committing whatever its size, and an MMA 10 more to issue: where a slab's MMAs take less, a stage holds two. (One
    // slab a stage: 296 cycles a slab at any BN up to 128. With a warp index the compiler cannot know to be uniform, 388.
    // With the loop inside a lane == 0 branch, 330 and 70 for each MMA.)
    if (rank == 0) {
      pdl_wait();                                                    // as above
      const uint32_t idesc = idesc_i8(2 * BM, sh.bn);
      const uint16_t mask = (uint16_t)(3u << leader);
      const uint64_t adesc0 = umma_desc_sw128(smem_u32(smem)), bdesc0 = umma_desc_sw128(smem_u32(smem) + sh.per * A_BYTES);
      int st = 0, it = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = first; t < sh.tiles.total && ok; t += step, ++it) {
        const int buf = it & 1;
        if (!mbar_wait(acc_empty + buf, ((it >> 1) & 1) ^ 1)) { fail(VG_ERR_MMA_WAIT); break; }
        tc_fence_after();
        const uint32_t acc = tmem + buf * PBN;
        for (int s = s0; s < s1; s += sh.per) {
          if (!mbar_wait(full + st, ph)) { fail(VG_ERR_TMA_WAIT); ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t a = adesc0 + (uint64_t)(st * (sh.stage >> 4)), b = bdesc0 + (uint64_t)(st * (sh.stage >> 4));
#pragma unroll
            for (int kk = 0; kk < BK / 32; ++kk) umma_i8_pair(acc, a + kk * 2, b + kk * 2, idesc, (s > s0 || kk) ? 1u : 0u);
            if (sh.per == 2 && s + 1 < s1) {
              const uint64_t a1 = a + (A_BYTES >> 4), b1 = b + (uint64_t)(sh.b_slab >> 4);
#pragma unroll
              for (int kk = 0; kk < BK / 32; ++kk) umma_i8_pair(acc, a1 + kk * 2, b1 + kk * 2, idesc, 1u);
            }
            umma_commit_pair(empty + st, mask);
            if (s + sh.per >= s1) umma_commit_pair(acc_full + buf, mask);
          }
          __syncwarp();
          if (++st == sh.stages) { st = 0; ph ^= 1; }
        }
      }
    }
  } else {
    pdl_wait();
    const uint32_t acc_empty0 = dsmem_map(smem_u32(acc_empty), leader);
    int it = 0;
    for (int t = first; t < sh.tiles.total; t += step, ++it) {
      const int buf = it & 1;
      int mi, ni;
      sh.tiles.at(t, mi, ni);
      const int n0 = ni * sh.bn, cols = min(sh.bn, p.N - n0);
      fetch_sx(p, sx, n0, cols);
      const OutWarp o(p, mi * 2 * BM + rank * BM + r, n0);
      have = __all_sync(0xffffffffu, mbar_wait(acc_full + buf, (it >> 1) & 1));
      if (!have) { fail(VG_ERR_MMA_WAIT); break; }
      tc_fence_after();
      if (SPLIT) break;
      const uint32_t acc = tmem + buf * PBN + ((uint32_t)(quarter * 32) << 16);
      store_tile<4>(p, o, acc, cols, sx, turn, 2);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty0 + buf * 8);
    }
  }
  __syncwarp();
  if (SPLIT) {
    int mi, ni;
    sh.tiles.at(first, mi, ni);
    const int n0 = ni * sh.bn, cols = min(sh.bn, p.N - n0);
    cluster_sync_all();                                              // every CTA's MMAs are done: the rings are free
    auto to_rank = [rank](int q) { return (uint32_t)(2 * q + rank); };
    if (warp >= 2) {
      if (have) send_partials(smem_u32(smem), tmem + ((uint32_t)(quarter * 32) << 16), cols, part, p.split, r, turn, 2, to_rank);
      else report_lost(lost, p.split, to_rank);
    }
    cluster_sync_all();
    if (warp >= 2 && !*lost) finish_partials<2>(p, smem, OutWarp(p, mi * 2 * BM + rank * BM + r, n0), sx, cols, part, p.split, r, turn, 2);
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);       // let copies and MMAs in flight end before the blocks do
  }
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

// Clusters of 1 .. 8 CTAs the device holds at once with one CTA per SM (clusters stay within a GPC, so 8 CTAs leave more
// SMs idle than 2). The runtime counts one CTA per SM for any kernel that allocates TMEM.
struct Room {
  int sms, clusters[MAX_SPLIT + 1];
};

// The attribute belongs to the device's copy of a kernel: set once per kernel and device.
int allow_smem(const void* kernel, int bytes, int dev, std::atomic<unsigned long long>& done) {
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load() & bit) return 0;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit);
  return (int)e;
}

const Room* room_of(int dev) {
  static Room rooms[64];
  static std::atomic<unsigned long long> known{0};
  static std::mutex mu;
  const unsigned long long bit = 1ull << (dev & 63);
  Room& room = rooms[dev & 63];
  if (known.load() & bit) return &room;
  std::lock_guard<std::mutex> lk(mu);
  if (known.load() & bit) return &room;
  if (cudaDeviceGetAttribute(&room.sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return nullptr;
  static std::atomic<unsigned long long> done{0};
  if (allow_smem(reinterpret_cast<const void*>(gemm_int8_pair_kernel<true>), P_SMEM, dev, done)) return nullptr;
  for (int size = 1; size <= MAX_SPLIT; ++size) {
    cudaLaunchAttribute a;
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = size;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size * 256);
    cfg.blockDim = dim3(P_THREADS);
    cfg.dynamicSmemBytes = P_SMEM;
    cfg.attrs = &a;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&room.clusters[size], gemm_int8_pair_kernel<true>, &cfg) != cudaSuccess) return nullptr;
  }
  known.fetch_or(bit);
  return &room;
}

// Token tile and K split of the pair form: the shape with the least estimated time (us), from tiles of 64 tokens up.
// Fitted to single rounds of 20 - 60 tiles at K = 6144 and 17408: a slab takes 0.157 us at 64 tokens (waiting and copying),
// 0.19 at 128, 0.30 at 256 (MMAs: 512 cycles and the epilogue's share); a launch 3.6 us and 6 ns a token of its tiles,
// 5 us more when partial sums travel. Splitting pays where there are few tiles and much K: 256 x 5120 x 17408 46.0 us
// whole with 256-token tiles, 28.6 with 96, 26.7 split three ways; at K = 6144 12.9 with 96, 16.3 split. Work and weight
// stream overlap, but not fully (128 x 34816 x 5120: 32.9 us in one token tile, 39 in two).
void choose_pair(int N, int K, int M, const Room& room, PairShape* sh, int* split) {
  const int slabs = (K + BK - 1) / BK, least = (N + PBN - 1) / PBN;
  const double weights = (double)M * K / 6.2e6;                 // from memory at 6.2 TB/s
  double best = 1e30;
  sh->tiles.mt = (M + 2 * BM - 1) / (2 * BM);
  for (int nt = least; nt <= min(4 * least, least + 6); ++nt) {
    const int bn = max(64, ((N + nt - 1) / nt + 31) / 32 * 32);
    const int used = (N + bn - 1) / bn;
    const double slab = max(0.125 + 0.0005 * bn, 0.00117 * bn);
    for (int s = 1; s <= PAIR_MAX_SPLIT && s <= max(1, slabs / 4); ++s) {
      const double rounds = ceil((double)sh->tiles.mt * used / max(1, room.clusters[2 * s]));
      const double work = rounds * ((slabs + s - 1) / s) * slab, fixed = 3.6 + 0.006 * bn;
      const double t = max(work, weights) + 0.2 * min(work, weights) + (s > 1 ? rounds * (fixed + 4.0 + 0.5 * s) : fixed);
      if (t < best) {
        best = t;
        sh->bn = bn;
        sh->tiles.nt = used;
        *split = s;
      }
    }
  }
  sh->b_slab = sh->bn / 2 * BK;
  sh->per = sh->bn < 160 ? 2 : 1;
  sh->stage = sh->per * (A_BYTES + sh->b_slab);
  sh->stages = min(P_MAX_STAGES, P_RING / sh->stage);
}

template <bool SPLIT>
int launch_pair(const I8Params& p, const PairShape& sh, int sms, int dev, const CUtensorMap& tw, const CUtensorMap& tx, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  const int rc = allow_smem(reinterpret_cast<const void*>(gemm_int8_pair_kernel<SPLIT>), P_SMEM, dev, done);
  if (rc) return rc;
  const int pairs = SPLIT ? sh.tiles.total * p.split : min(sms / 2, sh.tiles.total);
  return (int)launch_pdl_cluster(gemm_int8_pair_kernel<SPLIT>, dim3(2 * pairs), dim3(P_THREADS), SPLIT ? 2u * p.split : 2u, P_SMEM, st, p,
                                 sh, tw, tx);
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
  const Room* room = room_of(dev);
  if (!room) return -3;
  I8Params p{};
  p.sx = sx; p.sw = sw; p.out = out; p.ldo = ldo; p.M = M; p.N = N; p.K = K; p.split = 1; p.out_f32 = out_f32; p.err = err;
  const int es = out_f32 ? 4 : 2;
  p.vec = M % 4 == 0 && (N == 1 || ldo % 4 == 0) && reinterpret_cast<uintptr_t>(out) % (4 * es) == 0;
  const int slabs = (K + BK - 1) / BK;
  CUtensorMap tw, tx;
  int rc = make_map(codes, M, K, ldw, BM, &tw);
  if (rc) return rc;
  if (N <= NARROW_MAX) {
    const int bn = N <= 16 ? 16 : N <= 32 ? 32 : 64;
    const int tiles = (M + BM - 1) / BM;
    if (tiles > (1 << 26)) return -2;
    // The widest split whose clusters all run at once, two CTAs per SM, with four slabs per CTA at least. 16 x 5120 x
    // 17408 (40 tiles): 31.8 us unsplit, 20.6 / 19.5 / 17.3 with 2 / 3 / 6 parts, 23.1 with 7 (a second wave).
    for (int s = 2; s <= MAX_SPLIT && s <= slabs / 4; ++s)
      if (tiles <= 2 * room->clusters[s]) p.split = s;
    rc = make_map(q, N, K, ldq, bn, &tx);
    if (rc) return rc;
    switch (bn) {
      case 16: return launch<16>(p, dev, tw, tx, st);
      case 32: return launch<32>(p, dev, tw, tx, st);
      default: return launch<64>(p, dev, tw, tx, st);
    }
  }
  PairShape sh{};
  choose_pair(N, K, M, *room, &sh, &p.split);
  if ((long long)sh.tiles.mt * sh.tiles.nt > (1 << 26)) return -2;
  sh.tiles.total = sh.tiles.mt * sh.tiles.nt;
  rc = make_map(q, N, K, ldq, sh.bn / 2, &tx);
  if (rc) return rc;
  return p.split > 1 ? launch_pair<true>(p, sh, room->sms, dev, tw, tx, st) : launch_pair<false>(p, sh, room->sms, dev, tw, tx, st);
}
