// Mixture-of-experts products on the 5th-generation tensor cores (tcgen05 / TMEM / TMA), for more places than the few-token
// kernels of moe.cu take: h = silu(x Wg_e^T) * (x Wu_e^T) and y = h Wd_e^T over sorted rows.
//
// The weights are the 128-row M side of the MMA and the rows of one expert (a block of at most 256, as many as there are,
// in steps of 16) its N side: an expert's weights are read once for up to 256 tokens and little of an MMA is padding. Up to
// about 250 rows an expert the layer is bound by reading the weights, above it by the MMAs.
//   * up: the A tile is 64 gate and 64 up rows, alternating in groups of 8: one box of a 5-D tensor map over the
//     [expert][gate | up][row] layout. Gate and up values of one column of h then sit 8 lanes apart in one warp. B are the
//     expert's rows of xs, x sorted by a kernel before this one (gathered by TMA, four rows an instruction, the same kernel
//     took four times as long: one such instruction every 66 clocks).
//   * down: A is 128 rows of Wd, B the expert's consecutive rows of h. fp32 results per place go to y, and moe_combine sums
//     each token's places in their order.
// One persistent block an SM; warp 0 streams both operands through a ring of shared-memory stages across tiles, one lane of
// warp 1 issues the MMAs into one of two TMEM accumulators, warps 2-5 drain the other.
#include <algorithm>

#include "moe.cuh"
#include "tc_common.cuh"

namespace mmp {
namespace {

constexpr int MK = 64, MTHREADS = 192;

template <int STAGES>
struct MLayout {
  static constexpr int A_BYTES = 128 * MK * 2;
  static constexpr int B_BYTES = MOE_BLOCK_ROWS * MK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int BARS = STAGES * STAGE_BYTES;  // full[S], empty[S], acc_full[2], acc_empty[2]
  static constexpr int TMEM_SLOT = BARS + 8 * (2 * STAGES + 4);
  static constexpr int ABORT = TMEM_SLOT + 4;
  static constexpr int DYN = ABORT + 4 + 1024;
};

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int u, int v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];\n"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(u), "r"(v) : "memory");
}
template <bool UP, int STAGES>
__global__ void __launch_bounds__(MTHREADS, 1) moe_tc_kernel(const __grid_constant__ CUtensorMap tmA,
                                                             const __grid_constant__ CUtensorMap tmB, const MoeArgs A, int tiles) {
  using L = MLayout<STAGES>;
  extern __shared__ uint8_t dsmem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dsmem) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_addr(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int k_tiles = ((UP ? A.H : A.I) + MK - 1) / MK;
  auto full_bar = [&](int s) { return sbase + L::BARS + 8 * s; };
  auto empty_bar = [&](int s) { return sbase + L::BARS + 8 * (STAGES + s); };
  auto accf_bar = [&](int b) { return sbase + L::BARS + 8 * (2 * STAGES + b); };
  auto acce_bar = [&](int b) { return sbase + L::BARS + 8 * (2 * STAGES + 2 + b); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::ABORT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::TMEM_SLOT);

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf_bar(b), 1);
      mbar_init(acce_bar(b), 4);  // one elected lane per epilogue warp
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&tmA)) : "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&tmB)) : "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();
  const int nitems = __ldcg(&A.header->nblk) * tiles;

  int issued = 0;  // stages requested by warp 0 (drained at teardown after an abort)
  if (warp == 0) {
    int kc = 0;
    bool ok = true;
    for (int it = blockIdx.x; it < nitems && ok; it += gridDim.x) {
      const int4 blk = __ldcg(A.blocks + it / tiles);
      const int tile = it % tiles;
      // B rows come in boxes of 32; rows past the block's last are not read
      const int nb = (blk.z + 31) / 32;
      const uint32_t bytes = L::A_BYTES + nb * 32 * (MK * 2);
      for (int kt = 0; kt < k_tiles; ++kt, ++kc) {
        const int s = kc % STAGES;
        if (kc >= STAGES) {
          ok = mbar_wait(empty_bar(s), ((kc / STAGES) - 1) & 1, abort_flag, A.err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        const uint32_t a_s = sbase + s * L::STAGE_BYTES, b_s = a_s + L::A_BYTES;
        if (lane == 0) {
          mbar_expect_tx(full_bar(s), bytes);
          if (UP) tma_load_5d(a_s, &tmA, full_bar(s), kt * MK, 0, 0, tile * 8, blk.x);
          else tma_load_3d(a_s, &tmA, full_bar(s), kt * MK, tile * 128, blk.x);
        }
        __syncwarp();  // the bytes are announced before any of them can arrive
        if (lane < nb) tma_load_2d(b_s + lane * 32 * MK * 2, &tmB, full_bar(s), kt * MK, blk.y + lane * 32);
        ++issued;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      int kc = 0, tc = 0;
      for (int it = blockIdx.x; it < nitems && !*abort_flag; it += gridDim.x, ++tc) {
        const int4 blk = __ldcg(A.blocks + it / tiles);
        const uint32_t idesc = umma_idesc_mn(128, (blk.z + 15) / 16 * 16);
        const int buf = tc & 1;
        if (tc >= 2 && !mbar_wait(acce_bar(buf), ((tc >> 1) - 1) & 1, abort_flag, A.err)) break;
        tc_fence_after();
        bool ok = true;
        for (int kt = 0; kt < k_tiles; ++kt, ++kc) {
          const int s = kc % STAGES;
          if (!mbar_wait(full_bar(s), (kc / STAGES) & 1, abort_flag, A.err)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_s = sbase + s * L::STAGE_BYTES, b_s = a_s + L::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < MK / 16; ++kk)
            umma_f16(tmem + buf * 256, umma_desc(a_s + kk * 32), umma_desc(b_s + kk * 32), idesc, kt != 0 || kk != 0);
          umma_commit(empty_bar(s));
        }
        if (!ok) break;
        umma_commit(accf_bar(buf));
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3;  // TMEM lanes 32 q .. 32 q + 31
    int tc = 0;
    for (int it = blockIdx.x; it < nitems; it += gridDim.x, ++tc) {
      const int4 blk = __ldcg(A.blocks + it / tiles);
      const int tile = it % tiles;
      const int buf = tc & 1;
      bool ok = mbar_wait(accf_bar(buf), (tc >> 1) & 1, abort_flag, A.err);
      ok = __all_sync(0xffffffffu, ok && !*abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_lane = tmem + (static_cast<uint32_t>(q * 32) << 16) + buf * 256;
#pragma unroll 1
      for (int cb = 0; cb < blk.z; cb += 16) {
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
            if (c < blk.z && i < A.I) A.h[static_cast<int64_t>(blk.y + c) * A.I + i] = f2bf(gt / (1.f + __expf(-gt)) * uu);
          }
        } else {
          const int col = tile * 128 + q * 32 + lane;
          float* y = A.y + static_cast<int64_t>(blk.y + cb) * A.H + col;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (cb + j < blk.z && col < A.H) y[static_cast<int64_t>(j) * A.H] = __uint_as_float(v[j]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(acce_bar(buf)) : "memory");
    }
  }

  if (tid == 0 && *abort_flag) {
    for (int i = max(0, issued - STAGES); i < issued; ++i) mbar_drain(full_bar(i % STAGES), (i / STAGES) & 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
  }
}

int encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return mmp_set_error(MMP_ERR_INVALID, "mmp_moe_experts: tensor map encode failed (%d)", static_cast<int>(r));
  return MMP_OK;
}

template <bool UP>
int launch_products(const CUtensorMap& ma, const CUtensorMap& mb, const MoeArgs& A, int tiles, int max_blocks, int sms, cudaStream_t s) {
  constexpr int STAGES = 4;
  using L = MLayout<STAGES>;
  auto kern = moe_tc_kernel<UP, STAGES>;
  static bool set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::DYN);
    if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: shared memory attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  const int grid = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(max_blocks) * tiles, sms));
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
    const u64 dims[2] = {H, R}, strides[1] = {H * 2};
    const u32 box[2] = {MK, 32};
    if ((rc = encode(&mx, A.xs, 2, dims, strides, box)) != MMP_OK) return rc;
  }
  {
    const u64 dr = static_cast<u64>(A.d_r) * 2, de = A.E > 1 ? static_cast<u64>(A.d_e) * 2 : H * dr;
    const u64 dims[3] = {I, H, E}, strides[2] = {dr, de};
    const u32 box[3] = {MK, 128, 1};
    if ((rc = encode(&md, A.w_d, 3, dims, strides, box)) != MMP_OK) return rc;
  }
  {
    const u64 dims[2] = {I, R}, strides[1] = {I * 2};
    const u32 box[2] = {MK, 32};
    if ((rc = encode(&mh, A.h, 2, dims, strides, box)) != MMP_OK) return rc;
  }
  if ((rc = launch_products<true>(mgu, mx, A, (A.I + 63) / 64, max_blocks, sms, s)) != MMP_OK) return rc;
  if ((rc = launch_products<false>(md, mh, A, (A.H + 127) / 128, max_blocks, sms, s)) != MMP_OK) return rc;
  return mmp_check_launch("mmp_moe_experts");
}

}  // namespace mmp
