// Products of 8-bit operands with a power-of-two scale for each block of 128
// along the contracted axis, for sm_100a:
//   C[z, i, j] = sum_b 2^(ea[i, b] + eb[z, j, b]) sum_{k in block b} A[i, k] B[z, j, k]
//
// The tensor cores apply the scales themselves (tcgen05.mma, kind mxf8f6f4,
// block-scaled): a power-of-two scale per row and block is what they take, one
// byte each, so a block of 128 is four products of K = 32 that read the same
// scale byte, and the fp32 accumulator in tensor memory needs no second pass.
//
// Roles of a CTA's warps: 0 loads operand tiles by TMA into a ring of stages of
// one block of 128; 1 issues the products; 2 brings the scales (natural row
// order in memory) into the order of the tensor cores, four blocks at a time,
// from where warp 1 copies them to tensor memory; 4-7 read the accumulator,
// round and store it. Two accumulators alternate, so that the stores of one
// tile run under the products of the next.
//
// Measured: 16384 x 2560 x 10240 (pairs of CTAs) 313 us, 2.75 PFLOP/s, 0.83 of twice
// the measured bf16 rate; run back to back 363 us at the 1000 W power cap, 1.73
// times the bf16 library product's rate under the same cap. The tensor pipe is
// active 70 % of the time (78 % of the SMs' active cycles); without any operand
// loads the same kernel takes 278 us, without waiting for the previous tile's
// stores 301. 128 x 256 tiles of single CTAs 330 us.
#include "ss_ops.h"
#include "ss_quant.cuh"
#include "ss_tcgen05.cuh"

namespace mss {

static __device__ unsigned int g_fp8_err;

constexpr int kGemmM = 128;   // rows of A per tile
constexpr int kGemmK = 128;   // bytes of K per stage: one scale block
constexpr int kSfGroup = 4;   // scale blocks per copy (the bytes of one word)
constexpr int kSfSlots = 6;   // slots of a group's scales in shared memory
constexpr int kSfAhead = 3;   // groups under way behind the one handed over
// Two slots of 16 columns in tensor memory. The tensor cores execute one thread's
// copies and products in order, so a slot is written again only after the
// products that read it.
constexpr int kSfCols = 32;

struct GemmArgs {
  int rows_a, rows_b, batch, kb;  // kb: scale blocks
  int tiles_a, tiles_b, tiles;
  const uint8_t* a_scale;
  const uint8_t* b_scale;
  void* c;
  int tma_store;  // C may be stored by TMA (else through guarded stores)
  int words;      // scale rows may be read by 4-byte words
  int64_t a_scale_stride, b_scale_stride;  // bytes
  uint32_t polls;
};

template <int BN>
struct GemmCfg {
  static constexpr int kStageA = kGemmM * kGemmK;
  static constexpr int kStageB = BN * kGemmK;
  static constexpr int kStage = kStageA + kStageB;
  static constexpr int kSfBytes = 512 + (BN > 128 ? 1024 : 512);  // one group of both operands
  static constexpr int kOut = 4 * 4096;  // store staging: 32 rows x 128 bytes per warp
  static constexpr int kStages = BN >= 256 ? 4 : BN > 32 ? 5 : 8;
  static constexpr int kBytes = kStages * kStage + kOut + kSfSlots * kSfBytes + 512 + 1024;
  // accumulators: two of BN columns after the scales; for BN = 256 they share
  // columns (see the kernel)
  static constexpr int kTmem = 2 * BN + kSfCols > 256   ? 512
                               : 2 * BN + kSfCols > 128 ? 256
                               : 2 * BN + kSfCols > 64  ? 128
                                                        : 64;
  static constexpr int acc(int buf) { return buf == 0 ? kSfCols : (BN == 256 ? 256 : kSfCols + BN); }
};

// Waits for a phase of `bar`; false when it did not come within `polls` tries
// (recorded in the device error word) or when another role gave up.
__device__ __forceinline__ bool wait_role(uint64_t* bar, uint32_t parity, uint32_t polls,
                                          volatile int* gave_up) {
  for (uint32_t i = 0; i < polls; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*gave_up) return false;
  }
  *gave_up = 1;
  atomicOr(&g_fp8_err, kErrTmaTimeout);
  return false;
}

// Four scale bytes of blocks b .. b + 3 of a row, zero past the last block.
__device__ __forceinline__ uint32_t scale_word(const uint8_t* row, int b, int kb) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (b + e < kb) w |= static_cast<uint32_t>(__ldg(row + b + e)) << (8 * e);
  return w;
}

// Place in a ring of kN barriers: index and phase parity.
template <int kN>
struct Ring {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++at == kN) {
      at = 0;
      phase ^= 1;
    }
  }
};

// The scale order of the tensor cores: the word of row r of 128 (its bytes:
// four blocks) lies at byte (r % 32) * 16 + (r / 32) * 4. Rows past `rows` get
// zero bytes (their codes are zero-filled by the TMA). By 4-byte asynchronous
// copies where rows are whole words, so that a scale warp has several groups in
// flight; else through registers.
__device__ __forceinline__ void stage_scales(uint8_t* dst, const uint8_t* scales, int64_t stride,
                                             int64_t row0, int rows, int kb, int b, bool copies,
                                             int lane) {
  if (copies) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = q * 32 + lane;
      const bool in = r < rows;
      cp_async4(dst + lane * 16 + q * 4, scales + (in ? (row0 + r) * stride + b : 0), in);
    }
  } else {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = q * 32 + lane;
      w[q] = r < rows ? scale_word(scales + (row0 + r) * stride, b, kb) : 0u;
    }
    *reinterpret_cast<uint4*>(dst + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A scale warp: fills the ring of slots with the groups that `place` gives one after
// the other (false at the end): rows i0 .. of A, jt .. of batch z of B, block b. A group
// is handed over when kSfAhead younger ones are under way. The first slots are
// free from the start, so start() runs before the CTA's barriers are set up.
template <int BN, typename Place>
struct ScaleWarp {
  const GemmArgs& p;
  uint8_t* sf;
  const int slot_bytes;
  const bool copies;
  Place place;
  Ring<kSfSlots> at, out;
  int filled = 0, handed = 0;
  int i0 = 0, jt = 0, z = 0, b = 0;
  bool more = false;
  __device__ __forceinline__ ScaleWarp(const GemmArgs& p_, uint8_t* sf_, int bytes, bool copies_,
                                       Place place_)
      : p(p_), sf(sf_), slot_bytes(bytes), copies(copies_), place(place_) {}
  __device__ __forceinline__ void fill() {
    const int lane = threadIdx.x & 31;
    uint8_t* dst = sf + at.at * slot_bytes;
    const int64_t jrow = static_cast<int64_t>(z) * p.rows_b + jt;
    const int jrows = min(BN, p.rows_b - jt);
    stage_scales(dst, p.a_scale, p.a_scale_stride, i0, p.rows_a - i0, p.kb, b, copies, lane);
    stage_scales(dst + 512, p.b_scale, p.b_scale_stride, jrow, jrows, p.kb, b, copies, lane);
    if (BN > 128)
      stage_scales(dst + 1024, p.b_scale, p.b_scale_stride, jrow + 128, jrows - 128, p.kb, b,
                   copies, lane);
    cp_async_commit();
    at.next();
    ++filled;
    more = place(i0, jt, z, b);
  }
  __device__ __forceinline__ void start() {
    more = place(i0, jt, z, b);
    while (more && filled <= (copies ? kSfAhead : 0)) fill();
  }
  template <typename Arrive>
  __device__ __forceinline__ void hand_over(Arrive arrive) {
    fence_proxy_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) arrive(out.at);
    out.next();
    ++handed;
  }
  // wait(n, parity) waits for slot n to be free, arrive(n) hands it over.
  template <typename Wait, typename Arrive>
  __device__ __forceinline__ void run(Wait wait, Arrive arrive) {
    while (more) {
      cp_async_wait<kSfAhead>();
      hand_over(arrive);
      if (!__all_sync(0xffffffffu, wait(at.at, at.phase ^ 1))) break;
      fill();
    }
    cp_async_wait<0>();
    while (handed < filled) hand_over(arrive);
  }
};

// One warp's part of an accumulator tile: 32 rows (i0 ..) x BN columns (j0 ..) from
// tensor memory at src, rounded and stored through `stage` (4096 bytes).
// shared_last: start with the last columns, which the next tile's accumulator
// shares; `release` is called when those (or, with BN < 256, all) have been read.
template <int BN, typename OT, typename F>
__device__ __forceinline__ void store_tile(const GemmArgs& p, const CUtensorMap* map_c, int i0,
                                           int jt, int z, uint32_t src, uint8_t* stage,
                                           bool shared_last, F release) {
  const int lane = threadIdx.x & 31;
  constexpr int kCols = 128 / sizeof(OT);  // columns per 128-byte staging row
  constexpr int kChunks = BN / kCols;
  for (int q = 0; q < kChunks; ++q) {
    const int c = BN == 256 && shared_last ? kChunks - 1 - q : q;
    uint32_t w[32];  // one staging row: 32 words
    if constexpr (sizeof(OT) == 4) {
      tmem_ld32(src + c * kCols, w);
      tmem_ld_wait();
    } else {
      uint32_t f[32];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        tmem_ld32(src + c * kCols + h * 32, f);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e)
          w[h * 16 + e] = bf16x2_bits(__uint_as_float(f[2 * e]), __uint_as_float(f[2 * e + 1]));
      }
    }
    if (BN == 256 ? q == 0 : q == kChunks - 1) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) release();
    }
    if (p.tma_store && lane == 0) bulk_wait_read_all();
    __syncwarp();
    // 128-byte swizzle: 16-byte piece e of row l lies at piece e ^ (l % 8)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ (lane & 7)) << 4)) =
          make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
    const int j0 = jt + c * kCols;
    if (p.tma_store) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && i0 < p.rows_a && j0 < p.rows_b) {
        tma_store_3d(map_c, j0, i0, z, stage);
        bulk_commit();
      }
    } else {
      __syncwarp();
      OT* dst = static_cast<OT*>(p.c) + (static_cast<int64_t>(z) * p.rows_a + i0) * p.rows_b + j0;
      for (int r = 0; r < 32 && i0 + r < p.rows_a; ++r) {
#pragma unroll
        for (int e = 0; e < kCols / 32; ++e) {
          const int j = e * 32 + lane;
          const int byte = j * static_cast<int>(sizeof(OT));
          if (j0 + j < p.rows_b)
            dst[static_cast<int64_t>(r) * p.rows_b + j] = *reinterpret_cast<const OT*>(
                stage + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15));
        }
      }
      __syncwarp();
    }
  }
}

// One warp's part of a tile of few columns, stored transposed: out[j, i] for 32 rows
// i0 .. of A, one per lane.
template <int BN, typename OT, typename F>
__device__ __forceinline__ void store_tokens(const GemmArgs& p, int i0, int jt, uint32_t src,
                                             F release) {
  const int lane = threadIdx.x & 31;
  const int i = i0 + lane;
  OT* dst = static_cast<OT*>(p.c) + static_cast<int64_t>(jt) * p.rows_a + i;
  const int tokens = min(BN, p.rows_b - jt);
#pragma unroll
  for (int c = 0; c < BN; c += 16) {
    uint32_t w[16];
    tmem_ld16(src + c, w);
    tmem_ld_wait();
    if (c + 16 == BN) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) release();
    }
    if (i < p.rows_a) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (c + e < tokens)
          Elem<OT>::st(dst + static_cast<int64_t>(c + e) * p.rows_a, __uint_as_float(w[e]));
    }
  }
}

// kTokens: B has few rows, and C is stored transposed.
template <int BN, typename OT, bool kTokens>
__global__ void __launch_bounds__(256, 1)
    ss_fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_a,
                       const __grid_constant__ CUtensorMap map_b,
                       const __grid_constant__ CUtensorMap map_c, const GemmArgs p) {
  using Cfg = GemmCfg<BN>;
  constexpr int kStages = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* out_stage = smem + kStages * Cfg::kStage;
  uint8_t* sf = out_stage + Cfg::kOut;
  uint64_t* full = reinterpret_cast<uint64_t*>(sf + kSfSlots * Cfg::kSfBytes);
  uint64_t* empty = full + kStages;
  uint64_t* sf_full = empty + kStages;
  uint64_t* sf_empty = sf_full + kSfSlots;
  uint64_t* acc_full = sf_empty + kSfSlots;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drained = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // The loader's place: tile, block, ring. It starts on the empty ring at once,
  // while the other warps are still being set up.
  int ld_tile = blockIdx.x, ld_b = 0, fills = 0;
  int ld_i = 0, ld_j = 0, ld_z = 0;
  Ring<kStages> ld;
  auto load_block = [&] {
    if (ld_b == 0) {
      const int ta = ld_tile % p.tiles_a, tb = ld_tile / p.tiles_a;
      ld_i = ta * kGemmM;
      ld_j = tb % p.tiles_b * BN;
      ld_z = tb / p.tiles_b;
    }
    uint8_t* dst = smem + ld.at * Cfg::kStage;
    mbar_arrive_expect_tx(full + ld.at, Cfg::kStage);
    tma_load_2d(dst, &map_a, ld_b * kGemmK, ld_i, full + ld.at);
    tma_load_3d(dst + Cfg::kStageA, &map_b, ld_b * kGemmK, ld_j, ld_z, full + ld.at);
    ++fills;
    ld.next();
    if (++ld_b == p.kb) {
      ld_b = 0;
      ld_tile += gridDim.x;
    }
  };
  if (warp == 0 && elect_one()) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int s = 0; s < kSfSlots; ++s) {
      mbar_init(sf_full + s, 1);
      mbar_init(sf_empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full + s, 1);
      mbar_init(acc_empty + s, 4);
    }
    mbar_init(drained, 1);
    *gave_up = 0;
    fence_mbar_init();
    while (fills < kStages && ld_tile < p.tiles) load_block();
  }
  const int groups = (p.kb + kSfGroup - 1) / kSfGroup;
  int sf_tile = blockIdx.x, sf_group = 0;
  auto place = [&](int& i0, int& jt, int& z, int& b) {
    if (sf_tile >= p.tiles) return false;
    const int ta = sf_tile % p.tiles_a, tb = sf_tile / p.tiles_a;
    i0 = ta * kGemmM;
    jt = tb % p.tiles_b * BN;
    z = tb / p.tiles_b;
    b = sf_group * kSfGroup;
    if (++sf_group == groups) {
      sf_group = 0;
      sf_tile += gridDim.x;
    }
    return true;
  };
  ScaleWarp<BN, decltype(place)&> scales(p, sf, Cfg::kSfBytes, p.words != 0, place);
  if (warp == 2) scales.start();
  if (warp == 3) tmem_alloc<Cfg::kTmem>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      while (ld_tile < p.tiles && wait_role(empty + ld.at, ld.phase ^ 1, p.polls, gave_up))
        load_block();
      // nothing may land in this CTA's shared memory after its end
      for (int f = max(0, fills - kStages); f < fills; ++f)
        mbar_wait_bounded(full + f % kStages, (f / kStages) & 1);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = idesc_mxf8(kGemmM, BN);
      const uint64_t da0 = desc_swizzled(smem_u32(smem)), db0 = da0 + (Cfg::kStageA >> 4);
      int t = 0, to = 0;
      Ring<kStages> r;
      Ring<kSfSlots> g;
      // Copies a group's scales to tensor memory, one group ahead of the products
      // that need them, so that these do not wait for it.
      auto copy_scales = [&]() -> bool {
        if (!wait_role(sf_full + g.at, g.phase, p.polls, gave_up)) return false;
        tc_fence_after();
        const uint32_t dst = tmem + to * 16;
        to ^= 1;
        const uint64_t src = desc_scales(smem_u32(sf + g.at * Cfg::kSfBytes));
        tmem_copy_scales(dst, src);
        tmem_copy_scales(dst + 4, src + (512 >> 4));
        if (BN > 128) tmem_copy_scales(dst + 8, src + (1024 >> 4));
        mma_commit(sf_empty + g.at);
        g.next();
        return true;
      };
      int slot = 0;  // of the current group's scales
      bool ok = static_cast<int>(blockIdx.x) < p.tiles ? copy_scales() : true;
      for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x, ++t) {
        // BN = 256: two accumulators and the scales do not fit side by side, so the
        // accumulators share columns; the products of a tile wait until the
        // previous tile's stores have read those (they read them first)
        const int buf = t & 1;
        if (BN == 256) {
          if (t >= 1) ok = wait_role(acc_empty + (buf ^ 1), ((t - 1) >> 1) & 1, p.polls, gave_up);
        } else {
          if (t >= 2) ok = wait_role(acc_empty + buf, ((t - 2) >> 1) & 1, p.polls, gave_up);
        }
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + Cfg::acc(buf);
        const bool last = tile + static_cast<int>(gridDim.x) >= p.tiles;
        for (int b = 0; b < p.kb; ++b, r.next()) {
          const int byte = b % kSfGroup;
          if (!wait_role(full + r.at, r.phase, p.polls, gave_up)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t step = static_cast<uint64_t>(r.at * (Cfg::kStage >> 4));
          const uint32_t id = idesc | scale_select(byte), sfa = tmem + slot * 16;
#pragma unroll
          for (int k = 0; k < kGemmK / 32; ++k)
            mma_mxf8(d, da0 + step + 2 * k, db0 + step + 2 * k, id, sfa, sfa + 4, (b | k) != 0);
          mma_commit(empty + r.at);
          const bool end = b + 1 == p.kb;
          if (byte == kSfGroup - 1 || end) slot ^= 1;
          // after a group's first products: the next group's scales
          if (byte == 0 && !(last && b + kSfGroup >= p.kb) && !copy_scales()) {
            ok = false;
            break;
          }
        }
        if (ok) mma_commit(acc_full + buf);
      }
      // the tensor cores read shared memory and write tensor memory until here
      mma_commit(drained);
      mbar_wait_bounded(drained, 0);
    }
  } else if (warp == 2) {
    scales.run(
        [&](int n, uint32_t parity) { return wait_role(sf_empty + n, parity, p.polls, gave_up); },
        [&](int n) { mbar_arrive(sf_full + n); });
  } else if (warp >= 4) {
    const int quarter = warp & 3;  // lanes 32 quarter .. + 31 of tensor memory
    uint8_t* stage = out_stage + quarter * 4096;
    int t = 0;
    for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x, ++t) {
      const int ta = tile % p.tiles_a, tb = tile / p.tiles_a;
      const int z = tb / p.tiles_b, jb = tb % p.tiles_b;
      const int buf = t & 1;
      const bool ok = wait_role(acc_full + buf, (t >> 1) & 1, p.polls, gave_up);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t src = tmem + Cfg::acc(buf) + (static_cast<uint32_t>(quarter * 32) << 16);
      if constexpr (kTokens)
        store_tokens<BN, OT>(p, ta * kGemmM + quarter * 32, jb * BN, src,
                             [&] { mbar_arrive(acc_empty + buf); });
      else
        store_tile<BN, OT>(p, &map_c, ta * kGemmM + quarter * 32, jb * BN, z, src, stage, buf == 0,
                           [&] { mbar_arrive(acc_empty + buf); });
    }
    if (lane == 0) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 3) tmem_free<Cfg::kTmem>(tmem);
}

// ------------------------------------------------------------- pairs of CTAs
// The same product by pairs of CTAs on a 256 x 256 tile. One CTA's tile of 128 x 256
// reads and fills 24 KB of shared memory per 128 x 256 x 64 of product, more than
// the 128 bytes per clock that it has at full tensor rate; in a pair each CTA holds
// 128 rows of A and 128 of B, a third less for the same work. Each CTA loads its
// own operands and scales; a relay thread of rank 1 passes on to rank 0 that its
// stage is full, and one thread of rank 0 issues the products of both.
struct PairCfg {
  static constexpr int kStageA = kGemmM * kGemmK;
  static constexpr int kStage = 2 * kStageA;
  static constexpr int kSfBytes = 512 + 1024;
  static constexpr int kStages = 6;
  static constexpr int kOut = 4 * 4096;
  static constexpr int kBytes = kStages * kStage + kOut + kSfSlots * kSfBytes + 512 + 1024;
  static constexpr int kTmem = 512;
  static constexpr int acc(int buf) { return buf == 0 ? kSfCols : 256; }
};

// What the issuing thread has handed to the tensor cores, as its rings' next places: the
// arrivals that its commits make on each CTA's barriers.
struct Issued {
  uint32_t stages, groups, tiles;  // the rings': place, and phase from bit 8 on
};
template <int kN>
__device__ __forceinline__ uint32_t packed(const Ring<kN>& r) {
  return static_cast<uint32_t>(r.at) | (r.phase << 8);
}
// Waits for the last arrival on each of a ring's barriers (a barrier without one is ready).
__device__ __forceinline__ void drain_ring(uint64_t* bars, int n, uint32_t next) {
  const int at = static_cast<int>(next & 0xffu);
  const uint32_t phase = next >> 8;
  for (int s = 0; s < n; ++s) mbar_wait_bounded(bars + s, s < at ? phase : phase ^ 1);
}

// wait_role for barriers that the other CTA arrives at; giving up is told to it.
__device__ __forceinline__ bool wait_pair(uint64_t* bar, uint32_t parity, uint32_t polls,
                                          volatile int* gave_up, uint32_t other_flag) {
  for (uint32_t i = 0; i < polls; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*gave_up) return false;
  }
  *gave_up = 1;
  cluster_st32(other_flag, 1u);
  atomicOr(&g_fp8_err, kErrTmaTimeout);
  return false;
}

template <typename OT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(256, 1)
    ss_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_a,
                       const __grid_constant__ CUtensorMap map_b,
                       const __grid_constant__ CUtensorMap map_c, const GemmArgs p) {
  using Cfg = PairCfg;
  constexpr int kStages = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* out_stage = smem + kStages * Cfg::kStage;
  uint8_t* sf = out_stage + Cfg::kOut;
  uint64_t* full = reinterpret_cast<uint64_t*>(sf + kSfSlots * Cfg::kSfBytes);  // own copies
  uint64_t* other_full = full + kStages;  // rank 0: the other's stage, passed on
  uint64_t* empty = other_full + kStages;
  uint64_t* sf_full = empty + kStages;    // rank 0: both scale warps
  uint64_t* sf_empty = sf_full + kSfSlots;
  uint64_t* acc_full = sf_empty + kSfSlots;
  uint64_t* acc_empty = acc_full + 2;     // rank 0: both CTAs' store warps
  uint64_t* drained = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile Issued* issued = reinterpret_cast<volatile Issued*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  int ld_tile = pair, ld_b = 0, fills = 0;  // the loader's place, as above
  int ld_i = 0, ld_j = 0, ld_z = 0;
  Ring<kStages> ld;
  auto load_block = [&] {
    if (ld_b == 0) {
      const int ta = ld_tile % p.tiles_a, tb = ld_tile / p.tiles_a;
      ld_i = ta * 256 + rank * 128;
      ld_j = tb % p.tiles_b * 256 + rank * 128;
      ld_z = tb / p.tiles_b;
    }
    uint8_t* dst = smem + ld.at * Cfg::kStage;
    mbar_arrive_expect_tx(full + ld.at, Cfg::kStage);
    tma_load_2d(dst, &map_a, ld_b * kGemmK, ld_i, full + ld.at);
    tma_load_3d(dst + Cfg::kStageA, &map_b, ld_b * kGemmK, ld_j, ld_z, full + ld.at);
    ++fills;
    ld.next();
    if (++ld_b == p.kb) {
      ld_b = 0;
      ld_tile += pairs;
    }
  };
  if (warp == 0 && elect_one()) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(other_full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int s = 0; s < kSfSlots; ++s) {
      mbar_init(sf_full + s, 2);
      mbar_init(sf_empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full + s, 1);
      mbar_init(acc_empty + s, 8);
    }
    mbar_init(drained, 1);
    *gave_up = 0;
    fence_mbar_init();
    while (fills < kStages && ld_tile < p.tiles) load_block();
  }
  const int groups = (p.kb + kSfGroup - 1) / kSfGroup;
  int sf_tile = pair, sf_group = 0;
  auto place = [&](int& i0, int& jt, int& z, int& b) {
    if (sf_tile >= p.tiles) return false;
    const int ta = sf_tile % p.tiles_a, tb = sf_tile / p.tiles_a;
    i0 = ta * 256 + rank * 128;
    jt = tb % p.tiles_b * 256;
    z = tb / p.tiles_b;
    b = sf_group * kSfGroup;
    if (++sf_group == groups) {
      sf_group = 0;
      sf_tile += pairs;
    }
    return true;
  };
  ScaleWarp<256, decltype(place)&> scales(p, sf, Cfg::kSfBytes, p.words != 0, place);
  if (warp == 2) scales.start();
  __syncwarp();
  cluster_sync_all();  // both CTAs run and see the barriers
  if (warp == 3) tmem_alloc_pair<Cfg::kTmem>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t other_flag =
      cluster_map(smem_u32(const_cast<const int*>(gave_up)), static_cast<uint32_t>(rank ^ 1));
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return wait_pair(bar, parity, p.polls, gave_up, other_flag);
  };

  if (warp == 0) {
    if (elect_one()) {
      while (ld_tile < p.tiles && wait(empty + ld.at, ld.phase ^ 1)) load_block();
      // nothing may land in this CTA's shared memory after its end: neither
      // copies nor the arrivals of the products that read them
      for (int f = max(0, fills - kStages); f < fills; ++f) {
        mbar_wait_bounded(full + f % kStages, (f / kStages) & 1);
        if (!*gave_up) wait(empty + f % kStages, (f / kStages) & 1);
      }
    }
  } else if (warp == 1 && rank == 1) {
    if (elect_one()) {  // passes on that a stage is full
      const uint32_t to = cluster_map(smem_u32(other_full), 0);
      Ring<kStages> r;
      for (int tile = pair; tile < p.tiles && !*gave_up; tile += pairs) {
        for (int b = 0; b < p.kb; ++b, r.next()) {
          if (!wait(full + r.at, r.phase)) break;
          mbar_arrive_cluster(to + r.at * 8);
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = idesc_mxf8(256, 256);
      const uint64_t da0 = desc_swizzled(smem_u32(smem)), db0 = da0 + (Cfg::kStageA >> 4);
      int t = 0, to = 0;
      Ring<kStages> r;
      Ring<kSfSlots> g;
      Ring<2> done;
      auto copy_scales = [&]() -> bool {  // a group ahead, as above
        if (!wait(sf_full + g.at, g.phase)) return false;
        tc_fence_after();
        const uint32_t dst = tmem + to * 16;
        to ^= 1;
        const uint64_t src = desc_scales(smem_u32(sf + g.at * Cfg::kSfBytes));
        tmem_copy_scales_pair(dst, src);
        tmem_copy_scales_pair(dst + 4, src + (512 >> 4));
        tmem_copy_scales_pair(dst + 8, src + (1024 >> 4));
        mma_commit_pair(sf_empty + g.at);
        g.next();
        return true;
      };
      int slot = 0;
      bool ok = pair < p.tiles ? copy_scales() : true;
      for (int tile = pair; tile < p.tiles && ok; tile += pairs, ++t) {
        const int buf = t & 1;
        // the accumulators share columns (see the kernel above)
        if (t >= 1 && !wait(acc_empty + (buf ^ 1), ((t - 1) >> 1) & 1)) break;
        tc_fence_after();
        const uint32_t d = tmem + Cfg::acc(buf);
        const bool last = tile + pairs >= p.tiles;
        for (int b = 0; b < p.kb; ++b, r.next()) {
          const int byte = b % kSfGroup;
          if (!wait(full + r.at, r.phase) || !wait(other_full + r.at, r.phase)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t step = static_cast<uint64_t>(r.at * (Cfg::kStage >> 4));
          const uint32_t id = idesc | scale_select(byte), sfa = tmem + slot * 16;
#pragma unroll
          for (int k = 0; k < kGemmK / 32; ++k)
            mma_mxf8_pair(d, da0 + step + 2 * k, db0 + step + 2 * k, id, sfa, sfa + 4,
                          (b | k) != 0);
          mma_commit_pair(empty + r.at);
          const bool end = b + 1 == p.kb;
          if (byte == kSfGroup - 1 || end) slot ^= 1;
          if (byte == 0 && !(last && b + kSfGroup >= p.kb) && !copy_scales()) {
            ok = false;
            r.next();
            break;
          }
        }
        if (ok) {
          mma_commit_pair(acc_full + buf);
          done.next();
        }
      }
      mma_commit_pair_own(drained);
      mbar_wait_bounded(drained, 0);
      for (int q = 0; q < 2; ++q) {
        const uint32_t to = cluster_map(smem_u32(const_cast<Issued*>(issued)), q);
        cluster_st32(to, packed(r));
        cluster_st32(to + 4, packed(g));
        cluster_st32(to + 8, packed(done));
      }
    }
  } else if (warp == 2) {
    const uint32_t to = cluster_map(smem_u32(sf_full), 0);
    scales.run([&](int n, uint32_t parity) { return wait(sf_empty + n, parity); },
               [&](int n) { mbar_arrive_cluster(to + n * 8); });
    const int filled = scales.filled;
    bool ok = *gave_up == 0;
    // the copies' last arrivals
    for (int f = max(0, filled - kSfSlots); f < filled && ok; ++f)
      ok = __all_sync(0xffffffffu, wait(sf_empty + f % kSfSlots, (f / kSfSlots) & 1));
  } else if (warp >= 4) {
    const int quarter = warp & 3;
    uint8_t* stage = out_stage + quarter * 4096;
    int t = 0;
    for (int tile = pair; tile < p.tiles; tile += pairs, ++t) {
      const int ta = tile % p.tiles_a, tb = tile / p.tiles_a;
      const int z = tb / p.tiles_b, jb = tb % p.tiles_b;
      const int buf = t & 1;
      if (!__all_sync(0xffffffffu, wait(acc_full + buf, (t >> 1) & 1))) break;
      tc_fence_after();
      const uint32_t src = tmem + Cfg::acc(buf) + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t bar = cluster_map(smem_u32(acc_empty + buf), 0);
      store_tile<256, OT>(p, &map_c, ta * 256 + rank * 128 + quarter * 32, jb * 256, z, src, stage,
                          buf == 0, [&] { mbar_arrive_cluster(bar); });
    }
    if (lane == 0) bulk_wait_all();
  }
  tc_fence_before();
  cluster_sync_all();  // neither CTA leaves while the other's work reaches into it
  // After giving up (both know by now) the roles have not waited for the last arrivals of
  // the products and copies that were issued.
  if (*gave_up && threadIdx.x == 0) {
    drain_ring(empty, kStages, issued->stages);
    drain_ring(sf_empty, kSfSlots, issued->groups);
    drain_ring(acc_full, 2, issued->tiles);
  }
  if (warp == 3) tmem_free_pair<Cfg::kTmem>(tmem);
}

// ------------------------------------------- few rows of B (tokens), few tiles
// C transposed: out[j, i], j one of at most BN tokens, i a weight row, for weights of
// so few row tiles that one CTA per tile leaves SMs idle: the CTAs of a cluster
// cut K between them and add their partial sums in rank order through distributed
// shared memory. Bound by latency: launch, first bytes, the cluster's barriers.
template <int BN>
struct SkinnyCfg {
  static constexpr int kStageA = kGemmM * kGemmK;
  static constexpr int kStageB = BN * kGemmK;
  static constexpr int kStage = kStageA + kStageB;
  static constexpr int kStages = BN <= 32 ? 8 : BN <= 64 ? 6 : 5;
  static constexpr int kSfBytes = 1024;
  static constexpr int kBytes = kStages * kStage + kSfSlots * kSfBytes + 512 + 1024;
  static constexpr int kAcc = kSfCols;
  static constexpr int kTmem = BN + kAcc > 128 ? 256 : (BN + kAcc > 64 ? 128 : 64);
  static_assert(BN * kGemmM * 4 <= kStages * kStage, "partial sums fit the stages");
};

template <int BN, typename OT>
__global__ void __launch_bounds__(256)
    ss_fp8_skinny_kernel(const __grid_constant__ CUtensorMap map_a,
                         const __grid_constant__ CUtensorMap map_b, const GemmArgs p) {
  using Cfg = SkinnyCfg<BN>;
  constexpr int kStages = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sf = smem + kStages * Cfg::kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(sf + kSfSlots * Cfg::kSfBytes);
  uint64_t* empty = full + kStages;
  uint64_t* sf_full = empty + kStages;
  uint64_t* sf_empty = sf_full + kSfSlots;
  uint64_t* drained = sf_empty + kSfSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank()), splits = static_cast<int>(cluster_size());
  const int ta = blockIdx.x / splits, jb = blockIdx.y;
  // this CTA's scale blocks, whole groups where each CTA gets several
  const int unit = p.kb >= 2 * kSfGroup * splits ? kSfGroup : 1;
  const int units = (p.kb + unit - 1) / unit;
  const int b0 = units * rank / splits * unit;
  const int b1 = min(p.kb, units * (rank + 1) / splits * unit);
  int ld_b = b0, fills = 0;  // the loader's place, as above
  Ring<kStages> ld;
  auto load_block = [&] {
    uint8_t* dst = smem + ld.at * Cfg::kStage;
    mbar_arrive_expect_tx(full + ld.at, Cfg::kStage);
    tma_load_2d(dst, &map_a, ld_b * kGemmK, ta * kGemmM, full + ld.at);
    tma_load_3d(dst + Cfg::kStageA, &map_b, ld_b * kGemmK, jb * BN, 0, full + ld.at);
    ++fills;
    ++ld_b;
    ld.next();
  };
  if (warp == 0 && elect_one()) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int s = 0; s < kSfSlots; ++s) {
      mbar_init(sf_full + s, 1);
      mbar_init(sf_empty + s, 1);
    }
    mbar_init(drained, 1);
    *gave_up = 0;
    fence_mbar_init();
    while (fills < kStages && ld_b < b1) load_block();
  }
  int sf_next = b0;
  auto place = [&](int& i0, int& jt, int& z, int& b) {
    i0 = ta * kGemmM;
    jt = jb * BN;
    z = 0;
    b = sf_next;
    sf_next += kSfGroup;
    return b < b1;
  };
  ScaleWarp<BN, decltype(place)&> scales(p, sf, Cfg::kSfBytes,
                                         p.words != 0 && b0 % kSfGroup == 0, place);
  if (warp == 2) scales.start();
  if (warp == 3) tmem_alloc<Cfg::kTmem>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      while (ld_b < b1 && wait_role(empty + ld.at, ld.phase ^ 1, p.polls, gave_up)) load_block();
      for (int f = max(0, fills - kStages); f < fills; ++f)
        mbar_wait_bounded(full + f % kStages, (f / kStages) & 1);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = idesc_mxf8(kGemmM, BN);
      const uint64_t da0 = desc_swizzled(smem_u32(smem)), db0 = da0 + (Cfg::kStageA >> 4);
      const uint32_t d = tmem + Cfg::kAcc;
      uint32_t sfa = 0;
      Ring<kStages> r;
      Ring<kSfSlots> g;
      for (int f = 0; f < b1 - b0; ++f, r.next()) {
        const int byte = f % kSfGroup;
        if (byte == 0) {
          if (!wait_role(sf_full + g.at, g.phase, p.polls, gave_up)) break;
          tc_fence_after();
          sfa = tmem + (f / kSfGroup & 1) * 16;
          const uint64_t src = desc_scales(smem_u32(sf + g.at * Cfg::kSfBytes));
          tmem_copy_scales(sfa, src);
          tmem_copy_scales(sfa + 4, src + (512 >> 4));
          mma_commit(sf_empty + g.at);
          g.next();
        }
        if (!wait_role(full + r.at, r.phase, p.polls, gave_up)) break;
        tc_fence_after();
        const uint64_t step = static_cast<uint64_t>(r.at * (Cfg::kStage >> 4));
        const uint32_t id = idesc | scale_select(byte);
#pragma unroll
        for (int k = 0; k < kGemmK / 32; ++k)
          mma_mxf8(d, da0 + step + 2 * k, db0 + step + 2 * k, id, sfa, sfa + 4, (f | k) != 0);
        mma_commit(empty + r.at);
      }
      mma_commit(drained);
      mbar_wait_bounded(drained, 0);
    }
  } else if (warp == 2) {
    scales.run(
        [&](int n, uint32_t parity) { return wait_role(sf_empty + n, parity, p.polls, gave_up); },
        [&](int n) { mbar_arrive(sf_full + n); });
  }
  // warps 0 and 1 are past their last copy and product here
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  // partial sums as [token][weight row] in the operand stages
  float* part = reinterpret_cast<float*>(smem);
  const int quarter = warp & 3;
  const uint32_t src = tmem + Cfg::kAcc + (static_cast<uint32_t>(quarter * 32) << 16);
  for (int c = (warp >> 2) * 16; c < BN; c += 32) {
    uint32_t w[16];
    tmem_ld16(src + c, w);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e)
      part[(c + e) * kGemmM + quarter * 32 + lane] = __uint_as_float(w[e]);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 3) tmem_free<Cfg::kTmem>(tmem);
  cluster_sync_all();
  // four weight rows of a token per thread
  const int tokens = min(BN, p.rows_b - jb * BN);
  const uint32_t mine = smem_u32(part);
  const int i = (threadIdx.x & 31) * 4;
  const int row = ta * kGemmM + i;
  const bool whole = p.rows_a % 4 == 0 && (reinterpret_cast<uintptr_t>(p.c) & 15) == 0;
  for (int j = rank * 8 + (threadIdx.x >> 5); j < tokens; j += splits * 8) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (q < splits) {
        const float4 w = cluster_ld4(cluster_map(mine + (j * kGemmM + i) * 4, q));
        v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
      }
    }
    OT* dst = static_cast<OT*>(p.c) + static_cast<int64_t>(jb * BN + j) * p.rows_a + row;
    if (whole) {
      if (row < p.rows_a) {
        if constexpr (sizeof(OT) == 4)
          *reinterpret_cast<float4*>(dst) = v;
        else
          *reinterpret_cast<uint2*>(dst) = make_uint2(bf16x2_bits(v.x, v.y), bf16x2_bits(v.z, v.w));
      }
    } else {
      const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (row + q < p.rows_a) Elem<OT>::st(dst + q, e[q]);
    }
  }
  cluster_sync_all();  // no CTA leaves while another reads its sums
}

// ------------------------------------------------------------------ launches
static bool make_map(CUtensorMap* m, CUtensorMapDataType type, int rank, const void* base,
                     const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  auto fn = tensor_map_encoder();
  if (fn == nullptr) return false;
  const cuuint32_t one[3] = {1, 1, 1};
  return fn(m, type, rank, const_cast<void*>(base), dims, strides, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static bool operand_maps(const Fp8GemmParams& p, int bn, CUtensorMap* a, CUtensorMap* b) {
  const cuuint64_t da[2] = {static_cast<cuuint64_t>(p.k), static_cast<cuuint64_t>(p.rows_a)};
  const cuuint64_t sa[1] = {static_cast<cuuint64_t>(p.a_stride)};
  const cuuint32_t ba[2] = {kGemmK, kGemmM};
  const cuuint64_t db[3] = {static_cast<cuuint64_t>(p.k), static_cast<cuuint64_t>(p.rows_b),
                            static_cast<cuuint64_t>(p.batch)};
  const cuuint64_t sb[2] = {static_cast<cuuint64_t>(p.b_stride),
                            static_cast<cuuint64_t>(p.b_stride) * p.rows_b};
  const cuuint32_t bb[3] = {kGemmK, static_cast<cuuint32_t>(bn), 1};
  return make_map(a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.a, da, sa, ba) &&
         make_map(b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, p.b, db, sb, bb);
}

// Scale rows of whole words, the last one readable to its end.
static bool whole_words(const Fp8GemmParams& p) {
  const int64_t need = (p.k + 4 * kQBlock - 1) / (4 * kQBlock) * 4;
  return p.a_scale_stride % 4 == 0 && p.b_scale_stride % 4 == 0 && p.a_scale_stride >= need &&
         p.b_scale_stride >= need && (reinterpret_cast<uintptr_t>(p.a_scale) & 3) == 0 &&
         (reinterpret_cast<uintptr_t>(p.b_scale) & 3) == 0;
}

// BN columns per tile; pair: 256 x 256 tiles by pairs of CTAs (BN = 256).
template <int BN, typename OT, bool kPair = false, bool kTokens = false>
static cudaError_t gemm_go(const Fp8GemmParams& p, cudaStream_t stream) {
  CUtensorMap ma, mb, mc;
  if (!operand_maps(p, kPair ? 128 : BN, &ma, &mb)) return cudaErrorInvalidValue;
  GemmArgs g{};
  g.rows_a = p.rows_a;
  g.rows_b = p.rows_b;
  g.batch = p.batch;
  g.kb = (p.k + kQBlock - 1) / kQBlock;
  constexpr int kRows = kPair ? 256 : kGemmM;
  g.tiles_a = (p.rows_a + kRows - 1) / kRows;
  g.tiles_b = (p.rows_b + BN - 1) / BN;
  g.tiles = g.tiles_a * g.tiles_b * p.batch;
  g.a_scale = p.a_scale;
  g.b_scale = p.b_scale;
  g.c = p.c;
  g.polls = p.wait_polls;
  g.a_scale_stride = p.a_scale_stride;
  g.b_scale_stride = p.b_scale_stride;
  g.words = whole_words(p);
  const size_t pitch = static_cast<size_t>(p.rows_b) * sizeof(OT);
  g.tma_store = !kTokens && pitch % 16 == 0 && (reinterpret_cast<uintptr_t>(p.c) & 15) == 0;
  mc = ma;
  if (g.tma_store) {
    const cuuint64_t dc[3] = {static_cast<cuuint64_t>(p.rows_b), static_cast<cuuint64_t>(p.rows_a),
                              static_cast<cuuint64_t>(p.batch)};
    const cuuint64_t sc[2] = {pitch, pitch * p.rows_a};
    const cuuint32_t bc[3] = {static_cast<cuuint32_t>(128 / sizeof(OT)), 32, 1};
    if (!make_map(&mc,
                  sizeof(OT) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                  3, p.c, dc, sc, bc))
      return cudaErrorInvalidValue;
  }
  if constexpr (kPair) {
    auto fn = ss_fp8_pair_kernel<OT>;
    const cudaError_t e =
        cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg::kBytes);
    if (e != cudaSuccess) return e;
    fn<<<2 * std::min(g.tiles, sm_count() / 2), 256, PairCfg::kBytes, stream>>>(ma, mb, mc, g);
  } else {
    auto fn = ss_fp8_gemm_kernel<BN, OT, kTokens>;
    constexpr int kBytes = GemmCfg<BN>::kBytes;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) return e;
    fn<<<std::min(g.tiles, sm_count()), 256, kBytes, stream>>>(ma, mb, mc, g);
  }
  return cudaPeekAtLastError();
}

// Few rows of B: with row tiles for at least half the SMs one CTA each, the next
// tile's loads under this one's stores; with fewer, K is cut between CTAs: 32 x 5120
// x 2560 (20 tiles, 4 CTAs each) takes 8.3 us against 15.0 uncut; 32 x 2560 x 10240
// (80 tiles) 9.5 us uncut against 11.0 cut in two.
template <int BN, typename OT>
static cudaError_t skinny_go(const Fp8GemmParams& p, cudaStream_t stream) {
  using Cfg = SkinnyCfg<BN>;
  if ((p.rows_a + kGemmM - 1) / kGemmM * ((p.rows_b + BN - 1) / BN) * 2 > sm_count())
    return gemm_go<BN, OT, false, true>(p, stream);
  CUtensorMap ma, mb;
  if (!operand_maps(p, BN, &ma, &mb)) return cudaErrorInvalidValue;
  GemmArgs g{};
  g.rows_a = p.rows_a;
  g.rows_b = p.rows_b;
  g.kb = (p.k + kQBlock - 1) / kQBlock;
  g.tiles_a = (p.rows_a + kGemmM - 1) / kGemmM;
  g.tiles_b = (p.rows_b + BN - 1) / BN;
  g.a_scale = p.a_scale;
  g.b_scale = p.b_scale;
  g.c = p.c;
  g.polls = p.wait_polls;
  g.a_scale_stride = p.a_scale_stride;
  g.b_scale_stride = p.b_scale_stride;
  g.words = whole_words(p);
  // share K while every CTA still has an SM of its own and two blocks of 128
  int splits = 1;
  while (splits < 8 && g.tiles_a * g.tiles_b * splits * 2 <= sm_count() &&
         g.kb / (splits * 2) >= 2)
    splits *= 2;
  auto fn = ss_fp8_skinny_kernel<BN, OT>;
  const cudaError_t e =
      cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(g.tiles_a * splits, g.tiles_b, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = Cfg::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, ma, mb, g);
}

template <typename OT>
static cudaError_t gemm_any(const Fp8GemmParams& p, cudaStream_t stream) {
  if (p.transposed) {
    if (p.rows_b <= 16) return skinny_go<16, OT>(p, stream);
    if (p.rows_b <= 32) return skinny_go<32, OT>(p, stream);
    if (p.rows_b <= 64) return skinny_go<64, OT>(p, stream);
    return skinny_go<128, OT>(p, stream);
  }
  // The tile shape with the least waves x time of a tile. A block of 128 takes a
  // tile of 256 x 256 (a pair) 0.45 us, 128 x 256 0.48, 128 x 128 0.31, 128 x 64 0.22
  // where many tiles run; 1 us per wave for its ends.
  const int sms = sm_count();
  const int64_t kb = (p.k + kQBlock - 1) / kQBlock;
  auto cost = [&](int m, int n, int units, int64_t block) {
    const int64_t tiles = static_cast<int64_t>((p.rows_a + m - 1) / m) * ((p.rows_b + n - 1) / n) *
                          p.batch;
    return (tiles + units - 1) / units * (kb * block + 100);
  };
  const int64_t c[4] = {cost(256, 256, sms / 2, 45), cost(128, 256, sms, 48),
                        cost(128, 128, sms, 31), cost(128, 64, sms, 22)};
  switch (std::min_element(c, c + 4) - c) {
    case 0: return gemm_go<256, OT, true>(p, stream);
    case 1: return gemm_go<256, OT>(p, stream);
    case 2: return gemm_go<128, OT>(p, stream);
    default: return gemm_go<64, OT>(p, stream);
  }
}

cudaError_t launch_fp8_gemm(const Fp8GemmParams& p, int out_dtype, cudaStream_t stream) {
  return out_dtype == MSS_BF16 ? gemm_any<__nv_bfloat16>(p, stream) : gemm_any<float>(p, stream);
}

unsigned int take_fp8_device_error() {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_fp8_err, sizeof(v)) != cudaSuccess) return ~0u;
  cudaMemcpyToSymbol(g_fp8_err, &zero, sizeof(zero));
  return v;
}

}  // namespace mss
