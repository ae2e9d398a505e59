// Mixture-of-experts products on the 5th-generation tensor cores (tcgen05 / TMEM / TMA), for more places than the few-token
// kernels of moe_few.cu take: h = silu(x Wg_e^T) * (x Wu_e^T) and y = h Wd_e^T over sorted rows.
//
// The weights are the 128-row M side of the MMA and the rows of one expert (a block of at most 256, as many as there are,
// in steps of 16) its N side: an expert's weights are read once for up to 256 tokens and little of an MMA is padding. Up to
// about 250 rows an expert the layer is bound by HBM, above it by the MMAs.
//   * up: the A tile is 64 gate and 64 up rows, alternating in groups of 8: one box of a 5-D tensor map over the
//     [expert][gate | up][row] layout. Gate and up values of one column of h then sit 8 lanes apart in one warp. B are the
//     expert's tokens: gathered from x four rows at a time, or, where experts have many, boxes of xs, which a kernel before
//     this one sorts (26 us for 4096 tokens x 8 places).
//   * down: A is 128 rows of Wd, B the expert's consecutive rows of h. fp32 results per place go to y, and moe_combine sums
//     each token's places in their order.
// One persistent block an SM, two of them a pair on 256 weight rows (cta_group::2): each loads its own weights and half of the
// rows, so 64 columns of K take 32 KB an SM instead of 48. Warp 0 streams the weights, warps 6 and 7 (or 6) the rows
// through a ring of shared-memory stages across tiles, the leader's warp 1 issues the MMAs into one of two TMEM accumulators,
// warps 2-5 drain the other.
#include <algorithm>

#include "moe.cuh"
#include "tc_common.cuh"

namespace mmp {
namespace {

// A stage is SUB tiles of 64 columns of K: with one, the thread that issues the MMAs waits and commits twice as often (2 of 8 large
// experts, 4096 tokens: 1131 us instead of 1094).
constexpr int MK = 64, SUB = 2, MTHREADS = 256;

template <int STAGES, int ROWS>
struct MLayout {
  static constexpr int A_BYTES = SUB * 128 * MK * 2;                  // this block's 128 weight rows
  static constexpr int B_BYTES = SUB * ROWS / 2 * MK * 2;             // its half of the rows
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int BARS = STAGES * STAGE_BYTES;  // full[S], empty[S], acc_full[2], acc_empty[2]
  static constexpr int TMEM_SLOT = BARS + 8 * (2 * STAGES + 4);
  static constexpr int ABORT = TMEM_SLOT + 4;
  static constexpr int DYN = ABORT + 4 + 1024;
};

__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok));
  return ok != 0;
}
// TMA loads into this block's shared memory that complete on a barrier of either block of the pair (no multicast).
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];\n"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y) : "memory");
}
// four rows of a map whose box is one row high
__device__ __forceinline__ void pair_gather4(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int4 r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
      "[%1, {%3, %4, %5, %6, %7}], [%2];\n"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w) : "memory");
}
// Weights: ONCE where most experts have one row block, so that they are the first to leave L2 (777 tokens x 4 of 60 experts
// 199 -> 193 us; with several blocks an expert they are read again: 4096 tokens x 2 of 8 large experts 1078 -> 1106 us).
template <bool ONCE>
__device__ __forceinline__ void pair_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, uint64_t policy) {
  if constexpr (!ONCE) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];\n"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
    return;
  }
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint [%0], "
      "[%1, {%3, %4, %5}], [%2], %6;\n"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "l"(policy) : "memory");
}
template <bool ONCE>
__device__ __forceinline__ void pair_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int u, int v,
                                             uint64_t policy) {
  if constexpr (!ONCE) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
        "[%1, {%3, %4, %5, %6, %7}], [%2];\n"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(u), "r"(v) : "memory");
    return;
  }
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint [%0], "
      "[%1, {%3, %4, %5, %6, %7}], [%2], %8;\n"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(u), "r"(v), "l"(policy) : "memory");
}
// Operands by the low words of their descriptors (start address / 16), the rest of which is the same for all of them.
__device__ __forceinline__ void pair_mma(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 a, b;\nmov.b64 a, {%1, %3};\nmov.b64 b, {%2, %3};\nsetp.ne.b32 p, %5, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, p;\n}\n"
      ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate));
}
// arrives on the barrier at this offset in both blocks once the MMAs issued so far have completed
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
               ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

__device__ __forceinline__ void arrive_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(mapa(bar, 0)) : "memory");
}

// Work item `it`: a row block of an expert and a 256-row weight tile. The items of one tile over an expert's blocks follow
// one another, so that its weights come from HBM once (2 of 8 large experts, four blocks each: block by block their 117 MB
// would pass through L2 four times).
struct Item { int expert, row0, n, tile; };
__device__ __forceinline__ int4 moe_block(const MoeArgs& A, int it, int tiles, int nitems) {
  return __ldcg(A.blocks + min(it, nitems - 1) / tiles);  // past the last: not used
}
__device__ __forceinline__ Item moe_item(const MoeArgs& A, const int4& r, int it, int tiles) {
  const int b = it / tiles;
  const int nb = (r.z + A.block_rows - 1) / A.block_rows, q = it - (b - r.w) * tiles, tile = q / nb, j = q - tile * nb;
  // blocks of nearly equal size
  const int r0 = static_cast<int>(static_cast<int64_t>(r.z) * j / nb), r1 = static_cast<int>(static_cast<int64_t>(r.z) * (j + 1) / nb);
  return {r.x, r.y + r0, r1 - r0, tile};
}

// Two blocks of a cluster are a pair on one 256-row tile: each loads its 128 weight rows and half of the block's rows of B,
// the leader (rank 0) issues the MMAs for both (cta_group::2), each drains its own 128 rows of the accumulator.
template <bool UP, int STAGES, int ROWS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MTHREADS, 1)
    moe_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const MoeArgs A, int tiles) {
  using L = MLayout<STAGES, ROWS>;
  constexpr bool ONCE = ROWS == MOE_BLOCK_ROWS_FEW, GATHER = UP && moe_gathers(ROWS);
  constexpr int BOX = 64;  // rows of a TMA box of B
  auto half_rows = [](int n) { return (n + 15) / 16 * 8; };  // a block's half of the MMA's N rows
  auto box_count = [=](int n) { return (half_rows(n) + BOX - 1) / BOX; };
  extern __shared__ uint8_t dsmem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dsmem) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_addr(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(rank));
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int k_tiles = ((UP ? A.H : A.I) + SUB * MK - 1) / (SUB * MK);
  auto full_bar = [&](int s) { return sbase + L::BARS + 8 * s; };
  auto empty_bar = [&](int s) { return sbase + L::BARS + 8 * (STAGES + s); };
  auto accf_bar = [&](int b) { return sbase + L::BARS + 8 * (2 * STAGES + b); };
  auto acce_bar = [&](int b) { return sbase + L::BARS + 8 * (2 * STAGES + 2 + b); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::ABORT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::TMEM_SLOT);

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);   // the leader's announcement of both blocks' bytes (used in the leader alone)
      mbar_init(empty_bar(s), 1);  // the leader's commit
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf_bar(b), 1);
      mbar_init(acce_bar(b), 8);  // one lane of each epilogue warp of both blocks (used in the leader alone)
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&tmA)) : "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&tmB)) : "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::);
  }
  tc_fence_before();
  pair_sync();  // both blocks' barriers are set up and their TMEM is allocated
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Behind another kernel than the plan itself, the plan is complete: that kernel let this one start only after its own wait
  // for it. The weights' warp reads nothing else that a kernel wrote and starts at once.
  if (GATHER) pdl_wait();
  const int nitems = __ldcg(&A.header->nblk) * tiles;
  const int4 first = nitems > 0 ? moe_block(A, pair, tiles, nitems) : int4{};
  if (warp != 0) {
    pdl_wait();
    pdl_trigger();
  }

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t policy = evict_first_policy();
      int kc = 0;
      bool ok = true;
      int4 next = first;
      for (int it = pair; it < nitems && ok; it += npairs) {
        const Item blk = moe_item(A, next, it, tiles);
        next = moe_block(A, it + npairs, tiles, nitems);  // here long before it is used
        const int tile = blk.tile * 2 + static_cast<int>(rank);
        const uint32_t bytes = 2 * (128 + (GATHER ? half_rows(blk.n) : box_count(blk.n) * BOX)) * (SUB * MK * 2);
        for (int kt = 0; kt < k_tiles; ++kt, ++kc) {
          const int s = kc % STAGES;
          if (kc >= STAGES && !mbar_wait(empty_bar(s), ((kc / STAGES) - 1) & 1, abort_flag, A.err)) {
            ok = false;
            break;
          }
          const uint32_t bar = mapa(full_bar(s), 0);  // the leader's; bytes may arrive there before they are announced
          if (rank == 0) mbar_expect_tx(full_bar(s), bytes);
          for (int j = 0; j < SUB; ++j) {
            const uint32_t a_s = sbase + s * L::STAGE_BYTES + j * 128 * MK * 2;
            const int k = (kt * SUB + j) * MK;  // zeros past K
            if (UP) pair_load_5d<ONCE>(a_s, &tmA, bar, k, 0, 0, tile * 8, blk.expert, policy);
            else pair_load_3d<ONCE>(a_s, &tmA, bar, k, tile * 128, blk.expert, policy);
          }
        }
      }
    }
    __syncwarp();
  } else if (GATHER && warp >= 6) {
    // Token rows by gathers of four; warp 6 takes the even ones, warp 7 the odd ones. Each has at least one in every stage: a
    // warp with nothing to load would not be held by the ring and fall a turn behind.
    static_assert(MTHREADS == 256, "two warps");
    int s = 0;
    uint32_t phase = 1;
    bool ok = true;
    static_assert(!GATHER || ROWS / 16 * 4 == 32, "a lane finds the token of one row");
    auto place = [&](const Item& blk) {  // past the last: the first, whose column of the accumulator is not used
      const int half = half_rows(blk.n), g = warp - 6 + lane / 4 * 2, r = static_cast<int>(rank) * half + g * 4 + lane % 4;
      return __ldcg(A.rows + blk.row0 + (g < half / 4 && r < blk.n ? r : 0));
    };
    int4 next = first;
    int mine = pair < nitems ? place(moe_item(A, next, pair, tiles)) : 0;
    for (int it = pair; it < nitems && ok; it += npairs) {
      const int gathers = half_rows(moe_item(A, next, it, tiles).n) / 4, token = mine / A.places;
      next = moe_block(A, it + npairs, tiles, nitems);
      int4 tok[ROWS / 16];
#pragma unroll
      for (int i = 0; i < ROWS / 16; ++i)
        tok[i] = make_int4(__shfl_sync(0xffffffffu, token, 4 * i), __shfl_sync(0xffffffffu, token, 4 * i + 1),
                           __shfl_sync(0xffffffffu, token, 4 * i + 2), __shfl_sync(0xffffffffu, token, 4 * i + 3));
      for (int kt = 0; kt < k_tiles && ok; ++kt) {
        ok = __all_sync(0xffffffffu, mbar_try(empty_bar(s), phase) || mbar_wait(empty_bar(s), phase, abort_flag, A.err));
        if (!ok) break;
        const uint32_t bar = mapa(full_bar(s), 0), b_s = sbase + s * L::STAGE_BYTES + L::A_BYTES;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < ROWS / 16; ++i)
            if (warp - 6 + 2 * i < gathers)
#pragma unroll
              for (int j = 0; j < SUB; ++j)
                pair_gather4(b_s + (j * ROWS / 2 + (warp - 6 + 2 * i) * 4) * MK * 2, &tmB, bar, (kt * SUB + j) * MK, tok[i]);
        }
        __syncwarp();
        if (kt == 0 && it + npairs < nitems) mine = place(moe_item(A, next, it + npairs, tiles));
        if (++s == STAGES) {
          s = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 6) {
    if (lane == 0) {
      int kc = 0;
      bool ok = true;
      int4 next = first;
      for (int it = pair; it < nitems && ok; it += npairs) {
        const Item blk = moe_item(A, next, it, tiles);
        next = moe_block(A, it + npairs, tiles, nitems);
        // this block's half of the MMA's N rows, in boxes of 64 (what lies past it is not read; boxes of 32 or 16
        // copy less and cost 6 and 20 % more where the MMAs bound the kernel: each box is an instruction)
        const int nb = box_count(blk.n), row = blk.row0 + static_cast<int>(rank) * half_rows(blk.n);
        for (int kt = 0; kt < k_tiles; ++kt, ++kc) {
          const int s = kc % STAGES;
          if (kc >= STAGES && !mbar_wait(empty_bar(s), ((kc / STAGES) - 1) & 1, abort_flag, A.err)) {
            ok = false;
            break;
          }
          const uint32_t bar = mapa(full_bar(s), 0), b_s = sbase + s * L::STAGE_BYTES + L::A_BYTES;
          for (int j = 0; j < SUB; ++j)
            for (int b = 0; b < nb; ++b)
              pair_load_2d(b_s + (j * ROWS / 2 + b * BOX) * MK * 2, &tmB, bar, (kt * SUB + j) * MK, row + b * BOX);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp walks through the stages and one lane issues: addresses then stay in uniform registers. In a branch of one
    // thread the four MMAs of 64 columns took 272 clocks to issue instead of 77, and the kernel was bound by that thread
    // (32 tokens x 2 of 8 large experts: 252 us instead of 231).
    if (rank == 0) {
      int s = 0, tc = 0;
      uint32_t phase = 0;
      const uint64_t desc = umma_desc(sbase);
      const uint32_t lo0 = static_cast<uint32_t>(desc), hi = static_cast<uint32_t>(desc >> 32);
      bool ok = true;
      int4 next = first;
      for (int it = pair; it < nitems && ok; it += npairs, ++tc) {
        const uint32_t idesc = umma_idesc_mn(256, half_rows(moe_item(A, next, it, tiles).n) * 2);
        next = moe_block(A, it + npairs, tiles, nitems);
        const int buf = tc & 1;
        ok = __all_sync(0xffffffffu, tc < 2 || mbar_wait(acce_bar(buf), ((tc >> 1) - 1) & 1, abort_flag, A.err));
        tc_fence_after();
        for (int kt = 0; kt < k_tiles && ok; ++kt) {
          ok = __all_sync(0xffffffffu, mbar_try(full_bar(s), phase) || mbar_wait(full_bar(s), phase, abort_flag, A.err));
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_lo = lo0 + s * (L::STAGE_BYTES >> 4), b_lo = a_lo + (L::A_BYTES >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < SUB * MK / 16; ++kk)
              pair_mma(tmem + buf * 256, a_lo + kk / 4 * (128 * MK * 2 >> 4) + kk % 4 * 2,
                       b_lo + kk / 4 * (ROWS / 2 * MK * 2 >> 4) + kk % 4 * 2, hi, idesc, kk != 0 || kt != 0);
            pair_commit(empty_bar(s));
          }
          __syncwarp();
          if (++s == STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
        if (ok && elect_one()) pair_commit(accf_bar(buf));
        __syncwarp();
      }
    }
    __syncwarp();
  } else if (warp < 6) {
    const int q = warp & 3;  // TMEM lanes 32 q .. 32 q + 31
    int tc = 0;
    for (int it = pair; it < nitems; it += npairs, ++tc) {
      const Item blk = moe_item(A, moe_block(A, it, tiles, nitems), it, tiles);
      const int tile = blk.tile * 2 + rank;
      const int buf = tc & 1;
      bool ok = mbar_wait(accf_bar(buf), (tc >> 1) & 1, abort_flag, A.err);
      ok = __all_sync(0xffffffffu, ok && !*abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_lane = tmem + (static_cast<uint32_t>(q * 32) << 16) + buf * 256;
#pragma unroll 1
      for (int cb = 0; cb < blk.n; cb += 16) {
        uint32_t v[16];
        tmem_ld16_nw(t_lane + cb, v);
        tmem_wait();
        if constexpr (UP) {
          // lane = (8 columns of h) x (gate, up) x 2: the gate lane finishes even rows, the up lane odd ones
          const int up = (lane >> 3) & 1;
          const int i = tile * 64 + (q * 2 + (lane >> 4)) * 8 + (lane & 7);
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float mine0 = __uint_as_float(v[j]), mine1 = __uint_as_float(v[j + 1]);
            const float got = __shfl_xor_sync(0xffffffffu, up ? mine0 : mine1, 8);
            const float gt = up ? got : mine0, uu = up ? mine1 : got;
            const int c = cb + j + up;
            // h is rounded to bf16, the type of the second product's operands
            if (c < blk.n && i < A.I) A.h[static_cast<int64_t>(blk.row0 + c) * A.I + i] = f2bf(silu(gt) * uu);
          }
        } else {
          const int col = tile * 128 + q * 32 + lane;
          float* y = A.y + static_cast<int64_t>(blk.row0 + cb) * A.H + col;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (cb + j < blk.n && col < A.H) y[static_cast<int64_t>(j) * A.H] = __uint_as_float(v[j]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader(acce_bar(buf));
    }
  }

  // teardown: after an abort copies may still be in flight to either block: the microseconds pass that they take
  if (tid == 0 && *abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < WAIT_BUDGET_CYCLES / 16) {
    }
  }
  tc_fence_before();
  __syncthreads();
  pair_sync();  // no block leaves while the other may still signal its barriers or read its operands
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
  }
  pair_sync();
}

int encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return mmp_set_error(MMP_ERR_INVALID, "mmp_moe_experts: tensor map encode failed (%d)", static_cast<int>(r));
  return MMP_OK;
}

template <bool UP, int STAGES, int ROWS>
int launch_products(const CUtensorMap& ma, const CUtensorMap& mb, const MoeArgs& A, int tiles, int max_blocks, int sms, cudaStream_t s) {
  using L = MLayout<STAGES, ROWS>;
  auto kern = moe_tc_kernel<UP, STAGES, ROWS>;
  static bool set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::DYN);
    if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: shared memory attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  const int grid = 2 * static_cast<int>(std::min<int64_t>(static_cast<int64_t>(max_blocks) * tiles, std::max(1, sms / 2)));
  cudaError_t e = launch_kind(1, kern, dim3(grid), dim3(MTHREADS), L::DYN, s, nullptr, 0, ma, mb, A, tiles);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  return MMP_OK;
}

}  // namespace

int moe_products_tc(const MoeArgs& A, int max_blocks, cudaStream_t s) {
  int rc = get_encoder();
  if (rc != MMP_OK) return rc;
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (sms <= 0) sms = 148;
  using u64 = cuuint64_t;
  using u32 = cuuint32_t;
  const u64 H = A.H, I = A.I, E = A.E, R = static_cast<u64>(A.T) * A.places;
  CUtensorMap mgu, mx, md, mh;
  {
    const u64 dims[5] = {H, 8, 2, I / 8, E};
    const u64 gr = static_cast<u64>(A.gu_r) * 2, ge = A.E > 1 ? static_cast<u64>(A.gu_e) * 2 : 2 * I * gr;
    const u64 strides[4] = {gr, I * gr, 8 * gr, ge};
    const u32 box[5] = {MK, 8, 2, 8, 1};
    if ((rc = encode(&mgu, A.w_gu, 5, dims, strides, box)) != MMP_OK) return rc;
  }
  {
    const bool gather = moe_gathers(A.block_rows);
    const u64 dims[2] = {H, gather ? static_cast<u64>(A.T) : R}, strides[1] = {(gather && A.T > 1 ? static_cast<u64>(A.x_t) : H) * 2};
    const u32 box[2] = {MK, gather ? 1u : 64u};
    if ((rc = encode(&mx, gather ? A.x : A.xs, 2, dims, strides, box)) != MMP_OK) return rc;
  }
  {
    const u64 dr = static_cast<u64>(A.d_r) * 2, de = A.E > 1 ? static_cast<u64>(A.d_e) * 2 : H * dr;
    const u64 dims[3] = {I, H, E}, strides[2] = {dr, de};
    const u32 box[3] = {MK, 128, 1};
    if ((rc = encode(&md, A.w_d, 3, dims, strides, box)) != MMP_OK) return rc;
  }
  {
    const u64 dims[2] = {I, R}, strides[1] = {I * 2};
    const u32 box[2] = {MK, 64};
    if ((rc = encode(&mh, A.h, 2, dims, strides, box)) != MMP_OK) return rc;
  }
  const int up = (A.I + 127) / 128, down = (A.H + 255) / 256;
  if (A.block_rows == MOE_BLOCK_ROWS_FEW) {
    if ((rc = launch_products<true, 4, MOE_BLOCK_ROWS_FEW>(mgu, mx, A, up, max_blocks, sms, s)) != MMP_OK) return rc;
    if ((rc = launch_products<false, 4, MOE_BLOCK_ROWS_FEW>(md, mh, A, down, max_blocks, sms, s)) != MMP_OK) return rc;
  } else {
    if ((rc = launch_products<true, 3, MOE_BLOCK_ROWS>(mgu, mx, A, up, max_blocks, sms, s)) != MMP_OK) return rc;
    if ((rc = launch_products<false, 3, MOE_BLOCK_ROWS>(md, mh, A, down, max_blocks, sms, s)) != MMP_OK) return rc;
  }
  return mmp_check_launch("mmp_moe_experts");
}

}  // namespace mmp
