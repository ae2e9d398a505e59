// Mixture-of-experts layer: top-k routing, the plan that sorts tokens by expert, the few-token products, the weighted sum.
//   route:   w_k = exp(l_k - max) / Z over the top_k largest logits (ties to the lowest index)
//   experts: h = silu(x Wg_e^T) * (x Wu_e^T);  out_t = addend_t + sum_k w_{t,k} Wd_e h_{t,k}
//
// With few tokens the layer is bound by reading each chosen expert's weights once, so the products stream weight rows from
// HBM straight into mma.m16n8k16 fragments (16 weight rows x 8 tokens): 16-byte loads, the k dimension permuted the same
// way in both operands so that a lane's 16 bytes are its fragments of two MMAs, no shared memory in front of them.
//   up:   a block takes 8 columns of h of one expert (8 gate + 8 up rows are the 16 MMA rows, so one thread ends with both
//         of a pair), its 8 warps split the k dimension and meet in shared memory;
//   down: a block takes 16 columns of the output for ALL experts, its warps take (expert, k range) tasks and leave 16 fp32
//         a place in shared memory, then sum each token's places in their order: no atomics, no partial results in HBM.
#include <algorithm>
#include <cooperative_groups.h>

#include "moe.cuh"

namespace cg = cooperative_groups;

namespace mmp {
namespace {

// ------------------------------------------------------------------------------------------------ routing
struct RouteParams {
  const void* logits; int64_t l_t;
  int T, E, top_k, renorm, shared;
  float* weights; int32_t* ids;  // [T, top_k + shared], contiguous
};

// Floats as unsigned integers of the same order; 0 stands for "not to be chosen" (-inf, NaN, already taken): every
// other float maps above it. +inf is the largest float: in fp32 the two tie; no bf16 is equal to it, there only the value
// is clamped.
constexpr float LARGEST = 3.402823466e38f;
template <bool F32>
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0u;
  if (F32) v = fminf(v, LARGEST);
  const uint32_t u = __float_as_uint(v + 0.f);  // + 0: the two zeros are one value
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return fminf(__uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k), LARGEST);
}

template <bool F32>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  if constexpr (F32) return static_cast<const float*>(p)[i];
  else return bf2f(static_cast<const bf16*>(p)[i]);
}

// One token by one warp; lane j ends with place j's expert and weight (j < top_k + shared). V values a lane. A bf16 key has
// 16 bits: with the index below it one maximum finds the largest key and, among equals, the lowest index.
template <int V, bool F32>
__device__ __forceinline__ void route_token(const RouteParams& P, int t, int lane, int& id, float& w) {
  const int64_t row = static_cast<int64_t>(t) * P.l_t;
  uint32_t key[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = lane + 32 * j;
    key[j] = e < P.E ? order_key<F32>(load_logit<F32>(P.logits, row + e)) : 0u;
  }
  float gate = 0.f;
  if (P.shared) gate = load_logit<F32>(P.logits, row + P.E);
  auto largest = [&]() {
    uint32_t m = key[0];
#pragma unroll
    for (int j = 1; j < V; ++j) m = max(m, key[j]);
    return __reduce_max_sync(0xffffffffu, m);
  };
  float z = 0.f;
  const uint32_t top = largest();
  const float vmax = key_value(top);
  if (!P.renorm) {
#pragma unroll
    for (int j = 0; j < V; ++j) z += key[j] ? expf(key_value(key[j]) - vmax) : 0.f;
    z = warp_sum(z);
  }
  id = -1;
  uint32_t mine = 0;
  if constexpr (F32) {
    uint32_t m = top;
    for (int k = 0; k < P.top_k && m; ++k) {  // m == 0: nothing left to choose
      int at = 1 << 30;
#pragma unroll
      for (int j = V - 1; j >= 0; --j) at = key[j] == m ? lane + 32 * j : at;
      at = __reduce_min_sync(0xffffffffu, at);
      if (lane == k) {
        id = at;
        mine = m;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = lane + 32 * j == at ? 0u : key[j];
      m = largest();
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = key[j] ? (key[j] & 0xffff0000u) | (0xffffu - (lane + 32 * j)) : 0u;
    for (int k = 0; k < P.top_k; ++k) {
      const uint32_t m = largest();
      if (m == 0) break;
      if (lane == k) {
        id = 0xffff - static_cast<int>(m & 0xffffu);
        // the low half of a bf16's key: 0, or all ones below zero
        mine = (m & 0xffff0000u) | ((m & 0x80000000u) ? 0u : 0xffffu);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = key[j] == m ? 0u : key[j];
    }
  }
  w = id >= 0 ? expf(key_value(mine) - vmax) : 0.f;
  if (P.renorm) z = warp_sum(w);
  if (id >= 0) w /= z;
  if (P.shared && lane == P.top_k) {
    id = P.E;
    w = 1.f / (1.f + expf(-gate));
  }
}

template <int V, bool F32>
__global__ void __launch_bounds__(256) moe_route_kernel(const RouteParams P) {
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= P.T) return;
  int id;
  float w;
  route_token<V, F32>(P, t, lane, id, w);
  const int n = P.top_k + P.shared;
  if (lane < n) {
    P.weights[static_cast<int64_t>(t) * n + lane] = w;
    P.ids[static_cast<int64_t>(t) * n + lane] = id;
  }
}

// ------------------------------------------------------------------------------------------------ plan
// Exclusive scan of one int2 a thread over a block of 1024 threads (x: rows, y: blocks or one for a live expert).
__device__ __forceinline__ int2 scan_block(int2 v, int2* warp_tot, int2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, s.x, o), b = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) {
      s.x += a;
      s.y += b;
    }
  }
  if (lane == 31) warp_tot[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int2 q = warp_tot[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, q.x, o), b = __shfl_up_sync(0xffffffffu, q.y, o);
      if (lane >= o) {
        q.x += a;
        q.y += b;
      }
    }
    warp_tot[lane] = q;
  }
  __syncthreads();
  total = warp_tot[31];
  const int2 before = warp > 0 ? warp_tot[warp - 1] : make_int2(0, 0);
  return make_int2(before.x + s.x - v.x, before.y + s.y - v.y);
}

// Expert of a place, -1 for none; an index outside the experts is reported and counts as none.
__device__ __forceinline__ int place_expert(const MoeArgs& A, int p, bool report) {
  const int t = p / A.places, k = p - t * A.places;
  const int e = A.ids[static_cast<int64_t>(t) * A.id_t + k];
  if (e < A.E) return e < 0 ? -1 : e;
  if (report) flag_error(A.err, DEVERR_INDEX);
  return -1;
}

// From an expert's row count (thread i has expert E - 1 - i: the last expert, which every token may share, comes first)
// to its record and, with `blocks`, its row blocks, written by the block that has `write`. Returns its first sorted row.
__device__ __forceinline__ int plan_expert(const MoeArgs& A, int e, int n, int2* warp_tot, bool blocks, bool write) {
  int2 total;
  const int nb = (n + MOE_BLOCK_ROWS - 1) / MOE_BLOCK_ROWS;
  const int2 pre = scan_block(make_int2(n, blocks ? nb : n > 0 ? 1 : 0), warp_tot, total);
  if (!write) return pre.x;
  if (blocks) {
    for (int b = 0; b < nb; ++b) A.blocks[pre.y + b] = make_int4(e, pre.x, n, b);
    if (threadIdx.x == 0) A.header->nblk = total.y;
  } else {
    if (n > 0) A.recs[pre.y] = make_int4(e, pre.x, n, 0);
    if (threadIdx.x == 0) A.header->nact = total.y;
  }
  return pre.x;
}

struct RouteAndPlan {
  MoeArgs A;
  RouteParams P;  // routed first where P.logits is set: P.weights / P.ids are A.weights / A.ids
};

// The whole plan in one block of 1024 threads, for at most MOE_FEW_PLACES places; V > 0: routing first.
template <int V, bool F32>
__global__ void __launch_bounds__(1024) moe_plan_few(const RouteAndPlan Q) {
  const MoeArgs& A = Q.A;
  __shared__ int cnt[MOE_MAX_EXPERTS];
  __shared__ int2 warp_tot[32];
  __shared__ short s_e[MOE_FEW_PLACES], s_rank[MOE_FEW_PLACES];
  pdl_trigger();  // the next kernel may start; it waits for this one's end before it reads the plan
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int R = A.T * A.places;
  for (int e = tid; e < A.E; e += 1024) cnt[e] = 0;
  if constexpr (V > 0) {
    for (int t = warp; t < A.T; t += 32) {
      int id;
      float w;
      route_token<V, F32>(Q.P, t, lane, id, w);
      if (lane < A.places) {
        Q.P.weights[t * A.places + lane] = w;
        Q.P.ids[t * A.places + lane] = id;
        s_e[t * A.places + lane] = static_cast<short>(id);
      }
    }
  } else {
    for (int p = tid; p < R; p += 1024) s_e[p] = static_cast<short>(place_expert(A, p, true));
  }
  __syncthreads();
  for (int p = tid; p < R; p += 1024) {
    const int e = s_e[p];
    if (e >= 0) s_rank[p] = static_cast<short>(atomicAdd(&cnt[e], 1));
  }
  __syncthreads();
  const int e = A.E - 1 - tid;
  const int off = plan_expert(A, e, e >= 0 ? cnt[e] : 0, warp_tot, false, true);
  __syncthreads();
  if (e >= 0) cnt[e] = off;
  __syncthreads();
  for (int p = tid; p < R; p += 1024) {
    const int q = s_e[p];
    const int r = q >= 0 ? cnt[q] + s_rank[p] : -1;
    if (q >= 0) A.rows[r] = p;
    A.pos[p] = r;
  }
}

// The plan of many places by one cluster: every block counts its share of the places in shared memory, reads the others'
// counts there (distributed shared memory), scans the experts for itself and scatters its share. One launch: counting,
// scanning and scattering as three took 16 us of 434 for 4096 tokens x 8 places.
constexpr int PLAN_BLOCKS = 8;

__global__ void __cluster_dims__(PLAN_BLOCKS, 1, 1) __launch_bounds__(1024) moe_plan_many(const MoeArgs A) {
  __shared__ int cnt[MOE_MAX_EXPERTS], at[MOE_MAX_EXPERTS];
  __shared__ int2 warp_tot[32];
  cg::cluster_group cluster = cg::this_cluster();
  const int me = static_cast<int>(cluster.block_rank()), tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();
  const int64_t R = static_cast<int64_t>(A.T) * A.places;
  const int p0 = static_cast<int>(R * me / PLAN_BLOCKS), p1 = static_cast<int>(R * (me + 1) / PLAN_BLOCKS);
  for (int e = tid; e < A.E; e += 1024) cnt[e] = 0;
  __syncthreads();
  for (int p = p0 + tid; p < p1; p += 1024) {
    const int e = place_expert(A, p, true);
    if (e >= 0) atomicAdd(&cnt[e], 1);
  }
  cluster.sync();
  const int e = A.E - 1 - tid;
  int n = 0, before = 0;
  if (e >= 0)
#pragma unroll
    for (int b = 0; b < PLAN_BLOCKS; ++b) {
      const int c = cluster.map_shared_rank(cnt, b)[e];
      n += c;
      before += b < me ? c : 0;
    }
  const int off = plan_expert(A, e, n, warp_tot, true, me == 0);
  if (e >= 0) at[e] = off + before;
  cluster.sync();  // no block leaves while its counts are read
  for (int p = p0 + tid; p < p1; p += 1024) {
    const int q = place_expert(A, p, false);
    const int r = q >= 0 ? atomicAdd(&at[q], 1) : -1;
    if (q >= 0) A.rows[r] = p;
    A.pos[p] = r;
  }
}

// Each token's row to the sorted rows of its places: block (token), read once, written once a place.
__global__ void __launch_bounds__(256) moe_sort_rows(const MoeArgs A) {
  pdl_wait();
  pdl_trigger();
  const int64_t t = blockIdx.x;
  for (int c = threadIdx.x * 8; c < A.H; c += 256 * 8) {
    const uint4 v = ld16(A.x + t * A.x_t + c);
    for (int k = 0; k < A.places; ++k) {
      const int r = A.pos[t * A.places + k];
      if (r >= 0) st16(A.xs + static_cast<int64_t>(r) * A.H + c, v);
    }
  }
}

// ------------------------------------------------------------------------------------------------ few-token products
__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_weight(const bf16* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 ld_rows(const bf16* p) { return __ldcg(reinterpret_cast<const uint4*>(p)); }

// 32-wide k chunks whose weights a warp holds in registers at once (2 rows x 4 x 16 bytes a lane). With 8 (two blocks of the
// up kernel an SM instead of three) 64 tokens x 8 of 256 experts (H 2048, I 512) took 265 us, with 4 they take 239.
constexpr int SLAB = 4;

// acc[f] (16 rows x 8 tokens) += W[16 rows, k] X[8 tokens, k]^T over the warp's k chunks c0, c0 + step, ... < c1. ra / rb:
// this lane's two weight rows (null: a row outside the matrix), xr[f]: this lane's token row of group f (null: none).
// keep: the weights of the only slab are in `a` already.
template <int NF>
__device__ __forceinline__ void warp_products(float (&acc)[NF][4], uint4 (&a)[SLAB][2], bool keep, const bf16* ra, const bf16* rb,
                                              const bf16* const (&xr)[NF], int c0, int c1, int step, int K, int t4) {
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int c = c0; c < c1; c += SLAB * step) {
    if (!keep || c != c0) {
#pragma unroll
      for (int j = 0; j < SLAB; ++j) {
        const int cc = c + j * step, k = cc * 32 + t4 * 8;
        const bool in = cc < c1 && k < K;
        a[j][0] = in && ra ? ld_weight(ra + k) : zero;
        a[j][1] = in && rb ? ld_weight(rb + k) : zero;
      }
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      uint4 b[SLAB];
#pragma unroll
      for (int j = 0; j < SLAB; ++j) {
        const int cc = c + j * step, k = cc * 32 + t4 * 8;
        b[j] = cc < c1 && k < K && xr[f] ? ld_rows(xr[f] + k) : zero;
      }
#pragma unroll
      for (int j = 0; j < SLAB; ++j) {
        mma_16816(acc[f], a[j][0].x, a[j][1].x, a[j][0].y, a[j][1].y, b[j].x, b[j].y);
        mma_16816(acc[f], a[j][0].z, a[j][1].z, a[j][0].w, a[j][1].w, b[j].z, b[j].w);
      }
    }
  }
}

constexpr int UP_WARPS = 8;

template <int NF>
__device__ __forceinline__ void up_pass(const MoeArgs& A, const int4 rec, int base, uint4 (&a)[SLAB][2], bool keep, const bf16* ra,
                                        const bf16* rb, int i0, float4* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const bf16* xr[NF];
  float acc[NF][4];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int n = base + f * 8 + g;
    xr[f] = n < rec.z ? A.x + static_cast<int64_t>(__ldcg(A.rows + rec.y + n) / A.places) * A.x_t : nullptr;
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[f][q] = 0.f;
  }
  warp_products<NF>(acc, a, keep, ra, rb, xr, warp, (A.H + 31) / 32, UP_WARPS, A.H, t4);
#pragma unroll
  for (int f = 0; f < NF; ++f) red[(warp * NF + f) * 32 + lane] = make_float4(acc[f][0], acc[f][1], acc[f][2], acc[f][3]);
  __syncthreads();
  for (int q = tid; q < NF * 32; q += UP_WARPS * 32) {
    float4 s = red[q];
#pragma unroll
    for (int w = 1; w < UP_WARPS; ++w) {
      const float4 v = red[w * NF * 32 + q];
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const int l = q & 31, n = base + (q >> 5) * 8 + (l & 3) * 2;
    bf16* dst = A.h + static_cast<int64_t>(rec.y + n) * A.I + i0 + (l >> 2);
    // h is rounded to bf16, the type of the second product's operands: half a step of 2^-8 relative, as the output's own
    if (n < rec.z) dst[0] = f2bf(s.x / (1.f + expf(-s.x)) * s.z);
    if (n + 1 < rec.z) dst[A.I] = f2bf(s.y / (1.f + expf(-s.y)) * s.w);
  }
  __syncthreads();
}

// Block (i, r): columns 8 i .. 8 i + 7 of h for the rows of the r-th live expert.
__global__ void __launch_bounds__(UP_WARPS * 32, 3) moe_up_few(const MoeArgs A) {
  __shared__ float4 red[UP_WARPS * 4 * 32];
  pdl_wait();
  pdl_trigger();  // after the wait: what the plan wrote is then visible to the next kernel before its own wait
  if (static_cast<int>(blockIdx.y) >= __ldcg(&A.header->nact)) return;
  const int4 rec = __ldcg(A.recs + blockIdx.y);
  const int lane = threadIdx.x & 31, g = lane >> 2, i0 = blockIdx.x * 8;
  const bf16* ra = A.w_gu + rec.x * A.gu_e + static_cast<int64_t>(i0 + g) * A.gu_r;
  const bf16* rb = ra + A.I * A.gu_r;
  const bool one = A.H <= SLAB * UP_WARPS * 32;  // the block's weights fit its registers: read once for any number of rows
  uint4 a[SLAB][2];
  int base = 0;
  if (rec.z <= 8) {
    up_pass<1>(A, rec, 0, a, false, ra, rb, i0, red);
  } else if (rec.z <= 16) {
    up_pass<2>(A, rec, 0, a, false, ra, rb, i0, red);
  } else {
    for (; base < rec.z; base += 32) up_pass<4>(A, rec, base, a, one && base > 0, ra, rb, i0, red);
  }
}

template <int NF>
__device__ __forceinline__ void down_pass(const MoeArgs& A, const int4 rec, int base, uint4 (&a)[SLAB][2], bool keep, const bf16* ra,
                                          const bf16* rb, int c0, int c1, float* val) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const bf16* xr[NF];
  float acc[NF][4];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int n = base + f * 8 + g;
    xr[f] = n < rec.z ? A.h + static_cast<int64_t>(rec.y + n) * A.I : nullptr;
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[f][q] = 0.f;
  }
  warp_products<NF>(acc, a, keep, ra, rb, xr, c0, c1, 1, A.I, t4);
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int n = base + f * 8 + t4 * 2;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (n + q < rec.z) {
        float* v = val + __ldcg(A.rows + rec.y + n + q) * 16;
        v[g] = acc[f][q];
        v[g + 8] = acc[f][q + 2];
      }
    }
  }
}

// Block b: output columns 16 b .. 16 b + 15 of every token. Tasks (expert, k range) over the warps.
template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 16 ? 1 : 2) moe_down_few(const MoeArgs A, int max_splits) {
  extern __shared__ float val[];  // [split][place][16]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int R = A.T * A.places, r0 = blockIdx.x * 16;
  // the plan is complete: the kernel before this one let it start only after its own wait for it
  const int nact = __ldcg(&A.header->nact);
  // fewer live experts than warps: several warps share an expert's k range
  const int splits = max(1, min(max_splits, WARPS / max(1, nact)));
  const int chunks = (A.I + 31) / 32, per = (chunks + splits - 1) / splits;
  uint4 a[SLAB][2];
  bool waited = false;
  for (int task = warp; task < nact * splits; task += WARPS) {
    const int sp = task % splits;
    const int4 rec = __ldcg(A.recs + task / splits);
    const int c0 = sp * per, c1 = min(chunks, c0 + per);
    const bf16* w = A.w_d + rec.x * A.d_e;
    const bf16* ra = r0 + g < A.H ? w + static_cast<int64_t>(r0 + g) * A.d_r : nullptr;
    const bf16* rb = r0 + 8 + g < A.H ? w + static_cast<int64_t>(r0 + 8 + g) * A.d_r : nullptr;
    if (!waited) {  // the first weights are requested while the kernel before this one still runs
#pragma unroll
      for (int j = 0; j < SLAB; ++j) {
        const int k = (c0 + j) * 32 + t4 * 8;
        const bool in = c0 + j < c1 && k < A.I;
        a[j][0] = in && ra ? ld_weight(ra + k) : make_uint4(0, 0, 0, 0);
        a[j][1] = in && rb ? ld_weight(rb + k) : make_uint4(0, 0, 0, 0);
      }
      pdl_wait();
    }
    const bool one = c1 - c0 <= SLAB;
    float* v = val + static_cast<int64_t>(sp) * R * 16;
    if (rec.z <= 8) {
      down_pass<1>(A, rec, 0, a, !waited, ra, rb, c0, c1, v);
    } else if (rec.z <= 16) {
      down_pass<2>(A, rec, 0, a, !waited, ra, rb, c0, c1, v);
    } else {
      for (int base = 0; base < rec.z; base += 32)
        down_pass<4>(A, rec, base, a, base == 0 ? !waited : one, ra, rb, c0, c1, v);
    }
    waited = true;
  }
  if (!waited) pdl_wait();
  pdl_trigger();
  __syncthreads();
  // each token's places in their order, two columns a thread
  for (int q = tid; q < A.T * 8; q += WARPS * 32) {
    const int t = q >> 3, c = (q & 7) * 2;
    if (r0 + c >= A.H) continue;
    float s0 = 0.f, s1 = 0.f;
    if (A.addend) {
      const float2 f = unpack_bf16x2(*reinterpret_cast<const uint32_t*>(A.addend + t * A.a_t + r0 + c));
      s0 = f.x;
      s1 = f.y;
    }
    for (int k = 0; k < A.places; ++k) {
      const int e = A.ids[t * A.id_t + k];
      if (e < 0 || e >= A.E) continue;
      const float w = A.weights[t * A.w_t + k];
      float y0 = 0.f, y1 = 0.f;
      for (int sp = 0; sp < splits; ++sp) {
        const float2 v = *reinterpret_cast<const float2*>(val + (static_cast<int64_t>(sp) * R + t * A.places + k) * 16 + c);
        y0 += v.x;
        y1 += v.y;
      }
      s0 = fmaf(w, y0, s0);
      s1 = fmaf(w, y1, s1);
    }
    *reinterpret_cast<uint32_t*>(A.out + t * A.o_t + r0 + c) = pack_bf16x2(s0, s1);
  }
}

// ------------------------------------------------------------------------------------------------ weighted sum
// out_t = addend_t + sum_k w_{t,k} y[pos_{t,k}]: block (token), eight columns a thread.
__global__ void __launch_bounds__(256) moe_combine(const MoeArgs A) {
  const int t = blockIdx.x;
  const int64_t tt = t;
  for (int c = threadIdx.x * 8; c < A.H; c += 256 * 8) {
    float s[8];
    if (A.addend) {
      const uint4 u = ld16(A.addend + tt * A.a_t + c);
      const float2 p0 = unpack_bf16x2(u.x), p1 = unpack_bf16x2(u.y), p2 = unpack_bf16x2(u.z), p3 = unpack_bf16x2(u.w);
      s[0] = p0.x; s[1] = p0.y; s[2] = p1.x; s[3] = p1.y; s[4] = p2.x; s[5] = p2.y; s[6] = p3.x; s[7] = p3.y;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = 0.f;
    }
#pragma unroll 4
    for (int k = 0; k < A.places; ++k) {
      const int r = A.pos[tt * A.places + k];
      if (r < 0) continue;
      const float w = A.weights[tt * A.w_t + k];
      const float4* y = reinterpret_cast<const float4*>(A.y + static_cast<int64_t>(r) * A.H + c);
      const float4 u = __ldcs(y), v = __ldcs(y + 1);
      s[0] = fmaf(w, u.x, s[0]); s[1] = fmaf(w, u.y, s[1]); s[2] = fmaf(w, u.z, s[2]); s[3] = fmaf(w, u.w, s[3]);
      s[4] = fmaf(w, v.x, s[4]); s[5] = fmaf(w, v.y, s[5]); s[6] = fmaf(w, v.z, s[6]); s[7] = fmaf(w, v.w, s[7]);
    }
    st16(A.out + tt * A.o_t + c, make_uint4(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]), pack_bf16x2(s[4], s[5]), pack_bf16x2(s[6], s[7])));
  }
}

// ------------------------------------------------------------------------------------------------ host side
template <template <int, bool> class F, typename... Args>
int by_width(int E, bool f32, Args&&... args) {
  if (E <= 64) return f32 ? F<2, true>::go(args...) : F<2, false>::go(args...);
  if (E <= 160) return f32 ? F<5, true>::go(args...) : F<5, false>::go(args...);
  if (E <= 256) return f32 ? F<8, true>::go(args...) : F<8, false>::go(args...);
  return f32 ? F<32, true>::go(args...) : F<32, false>::go(args...);
}

template <int V, bool F32>
struct LaunchRoute {
  static int go(const RouteParams& P, cudaStream_t s) {
    moe_route_kernel<V, F32><<<(P.T + 7) / 8, 256, 0, s>>>(P);
    return mmp_check_launch("mmp_moe_route");
  }
};
template <int V, bool F32>
struct LaunchPlan {
  static int go(const RouteAndPlan& Q, cudaStream_t s) {
    moe_plan_few<V, F32><<<1, 1024, 0, s>>>(Q);
    return mmp_check_launch("mmp_moe_layer");
  }
};

template <int WARPS>
int launch_down(const MoeArgs& A, cudaStream_t s) {
  const size_t one = static_cast<size_t>(A.T) * A.places * 64;
  const int splits = std::max(1, std::min<int>(WARPS, static_cast<int>(64 * 1024 / std::max<size_t>(1, one))));
  const size_t smem = one * splits;
  auto kern = moe_down_few<WARPS>;
  static bool set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MOE_FEW_PLACES * 64);
    if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: shared memory attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  cudaError_t e = launch_kind(1, kern, dim3((A.H + 15) / 16), dim3(WARPS * 32), smem, s, nullptr, 0, A, splits);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  return MMP_OK;
}

int few_products(const MoeArgs& A, cudaStream_t s) {
  const int R = A.T * A.places;
  cudaError_t e = launch_kind(1, moe_up_few, dim3(A.I / 8, std::min(R, A.E)), dim3(UP_WARPS * 32), 0, s, nullptr, 0, A);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  // 16 warps while one block an SM covers the columns, else two blocks of 8
  const int rc = (A.H + 15) / 16 <= 148 ? launch_down<16>(A, s) : launch_down<8>(A, s);
  return rc != MMP_OK ? rc : mmp_check_launch("mmp_moe_experts");
}

int many_products(const MoeArgs& A, const MoeLayout& L, cudaStream_t s) {
  cudaError_t e = launch_kind(1, moe_plan_many, dim3(PLAN_BLOCKS), dim3(1024), 0, s, nullptr, 0, A);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  e = launch_kind(1, moe_sort_rows, dim3(A.T), dim3(256), 0, s, nullptr, 0, A);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  const int rc = moe_products_tc(A, L.max_blocks, s);
  if (rc != MMP_OK) return rc;
  moe_combine<<<A.T, 256, 0, s>>>(A);
  return mmp_check_launch("mmp_moe_experts");
}

int check_route(const char* what, const void* logits, int dtype, int64_t l_t, int T, int E, int top_k, int shared) {
  if (T < 0 || E < 1 || E > MOE_MAX_EXPERTS || top_k < 1 || top_k > E || top_k + (shared ? 1 : 0) > MOE_MAX_TOPK)
    return mmp_set_error(MMP_ERR_INVALID, "%s: T=%d, %d experts, top_k %d: 1 <= top_k <= experts <= %d, at most %d places a token",
                         what, T, E, top_k, MOE_MAX_EXPERTS, MOE_MAX_TOPK);
  if (dtype != MMP_F32 && dtype != MMP_BF16) return mmp_set_error(MMP_ERR_INVALID, "%s: logits are fp32 or bf16", what);
  if (T > 0 && !logits) return mmp_set_error(MMP_ERR_INVALID, "%s: null logits", what);
  if (T > 1 && l_t < E + (shared ? 1 : 0)) return mmp_set_error(MMP_ERR_INVALID, "%s: logits rows overlap", what);
  return MMP_OK;
}

// Arguments shared by mmp_moe_experts and mmp_moe_layer.
int check_experts(const char* what, const MoeArgs& A, const void* workspace, size_t workspace_bytes, const MoeLayout& L) {
  if (A.H < 8 || A.H % 8 || A.I < 8 || A.I % 8 || A.H > (1 << 20) || A.I > (1 << 20))
    return mmp_set_error(MMP_ERR_INVALID, "%s: H=%d and I=%d must be positive multiples of 8", what, A.H, A.I);
  if (A.E < 1 || A.E > MOE_MAX_EXPERTS || A.places < 1 || A.places > MOE_MAX_TOPK)
    return mmp_set_error(MMP_ERR_INVALID, "%s: %d experts (at most %d), %d places a token (at most %d)", what, A.E, MOE_MAX_EXPERTS,
                         A.places, MOE_MAX_TOPK);
  if (static_cast<int64_t>(A.T) * A.places > (1 << 26))
    return mmp_set_error(MMP_ERR_INVALID, "%s: %d tokens of %d places are more than 2^26 places", what, A.T, A.places);
  if (A.T == 0) return MMP_OK;
  if (!A.x || !A.w_gu || !A.w_d || !A.out) return mmp_set_error(MMP_ERR_INVALID, "%s: null pointer", what);
  if (!aligned16(A.x) || !aligned16(A.w_gu) || !aligned16(A.w_d) || !aligned16(A.out) || !aligned16(A.addend) || A.x_t % 8 ||
      A.gu_e % 8 || A.gu_r % 8 || A.d_e % 8 || A.d_r % 8 || A.o_t % 8 || A.a_t % 8)
    return mmp_set_error(MMP_ERR_INVALID, "%s: rows must be 16-byte aligned", what);
  if ((A.T > 1 && (A.x_t < A.H || A.o_t < A.H || (A.addend && A.a_t < A.H))) || A.gu_r < A.H || A.d_r < A.I ||
      (A.E > 1 && (A.gu_e < 2 * A.I * A.gu_r || A.d_e < A.H * A.d_r)))
    return mmp_set_error(MMP_ERR_INVALID, "%s: rows or experts overlap", what);
  if (!workspace || workspace_bytes < L.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return mmp_set_error(MMP_ERR_INVALID, "%s: workspace of %zu bytes, 256-byte aligned, needed (%zu given)", what, L.bytes, workspace_bytes);
  return MMP_OK;
}

void place_workspace(MoeArgs& A, const MoeLayout& L, void* workspace) {
  char* w = static_cast<char*>(workspace);
  A.header = reinterpret_cast<MoeHeader*>(w + L.header);
  A.recs = reinterpret_cast<int4*>(w + L.recs);
  A.blocks = reinterpret_cast<int4*>(w + L.blocks);
  A.rows = reinterpret_cast<int*>(w + L.rows);
  A.pos = reinterpret_cast<int*>(w + L.pos);
  A.xs = reinterpret_cast<bf16*>(w + L.xs);
  A.h = reinterpret_cast<bf16*>(w + L.h);
  A.y = reinterpret_cast<float*>(w + L.y);
}

}  // namespace
}  // namespace mmp

using namespace mmp;

extern "C" int mmp_moe_route(const void* logits, int logits_dtype, int64_t l_t, int T, int E, int top_k, int renormalize,
                             int shared, float* weights, int32_t* ids, void* stream) {
  int rc = check_route("mmp_moe_route", logits, logits_dtype, l_t, T, E, top_k, shared);
  if (rc != MMP_OK || T == 0) return rc;
  if (!weights || !ids) return mmp_set_error(MMP_ERR_INVALID, "mmp_moe_route: null pointer");
  RouteParams P{logits, l_t, T, E, top_k, renormalize ? 1 : 0, shared ? 1 : 0, weights, ids};
  return by_width<LaunchRoute>(E, logits_dtype == MMP_F32, P, static_cast<cudaStream_t>(stream));
}

extern "C" size_t mmp_moe_workspace_size(int T, int places, int H, int I, int E) {
  if (T <= 0 || places <= 0 || H <= 0 || I <= 0 || E <= 0) return 0;
  return moe_layout(T, places, H, I, E).bytes;
}

extern "C" int mmp_moe_experts(const void* x, int64_t x_t, const void* w_gate_up, int64_t gu_e, int64_t gu_r, const void* w_down,
                               int64_t d_e, int64_t d_r, const float* weights, int64_t w_t, const int32_t* ids, int64_t id_t,
                               const void* addend, int64_t a_t, void* out, int64_t o_t, int T, int places, int H, int I, int E,
                               void* workspace, size_t workspace_bytes, int* err, void* stream) {
  if (T < 0) return mmp_set_error(MMP_ERR_INVALID, "mmp_moe_experts: T=%d", T);
  MoeArgs A{static_cast<const bf16*>(x), x_t, static_cast<const bf16*>(w_gate_up), gu_e, gu_r, static_cast<const bf16*>(w_down),
            d_e, d_r, weights, w_t, ids, id_t, static_cast<const bf16*>(addend), a_t, static_cast<bf16*>(out), o_t,
            T, places, H, I, E};
  A.err = err;
  const MoeLayout L = moe_layout(T, std::max(1, places), std::max(8, H), std::max(8, I), std::max(1, E));
  int rc = check_experts("mmp_moe_experts", A, workspace, workspace_bytes, L);
  if (rc != MMP_OK || T == 0) return rc;
  if (!weights || !ids || (T > 1 && (w_t < places || id_t < places)))
    return mmp_set_error(MMP_ERR_INVALID, "mmp_moe_experts: weights and ids must be [T, places]");
  place_workspace(A, L, workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (static_cast<int64_t>(T) * places > MOE_FEW_PLACES) return many_products(A, L, s);
  RouteAndPlan Q{A, {}};
  moe_plan_few<0, false><<<1, 1024, 0, s>>>(Q);
  return few_products(A, s);
}

extern "C" int mmp_moe_layer(const void* x, int64_t x_t, const void* logits, int logits_dtype, int64_t l_t, const void* w_gate_up,
                             int64_t gu_e, int64_t gu_r, const void* w_down, int64_t d_e, int64_t d_r, const void* addend,
                             int64_t a_t, void* out, int64_t o_t, int T, int top_k, int renormalize, int shared, int H, int I,
                             int E, void* workspace, size_t workspace_bytes, int* err, void* stream) {
  const int routed = E - (shared ? 1 : 0), places = top_k + (shared ? 1 : 0);
  int rc = check_route("mmp_moe_layer", logits, logits_dtype, l_t, T, routed, top_k, shared);
  if (rc != MMP_OK) return rc;
  MoeArgs A{static_cast<const bf16*>(x), x_t, static_cast<const bf16*>(w_gate_up), gu_e, gu_r, static_cast<const bf16*>(w_down),
            d_e, d_r, nullptr, places, nullptr, places, static_cast<const bf16*>(addend), a_t, static_cast<bf16*>(out), o_t,
            T, places, H, I, E};
  A.err = err;
  const MoeLayout L = moe_layout(T, places, std::max(8, H), std::max(8, I), std::max(1, E));
  rc = check_experts("mmp_moe_layer", A, workspace, workspace_bytes, L);
  if (rc != MMP_OK || T == 0) return rc;
  place_workspace(A, L, workspace);
  float* w = reinterpret_cast<float*>(static_cast<char*>(workspace) + L.weights);
  int32_t* ids = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + L.ids);
  A.weights = w;
  A.ids = ids;
  RouteParams P{logits, l_t, T, routed, top_k, renormalize ? 1 : 0, shared ? 1 : 0, w, ids};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (static_cast<int64_t>(T) * places <= MOE_FEW_PLACES) {
    rc = by_width<LaunchPlan>(routed, logits_dtype == MMP_F32, RouteAndPlan{A, P}, s);
    return rc != MMP_OK ? rc : few_products(A, s);
  }
  rc = by_width<LaunchRoute>(routed, logits_dtype == MMP_F32, P, s);
  return rc != MMP_OK ? rc : many_products(A, L, s);
}
