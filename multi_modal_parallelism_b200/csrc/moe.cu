// Mixture-of-experts layer: top-k routing, the plan that sorts tokens by expert, the few-token products, the weighted sum.
//   route:   w_k = exp(l_k - max) / Z over the top_k largest logits (ties to the lowest index)
//   experts: h = silu(x Wg_e^T) * (x Wu_e^T);  out_t = addend_t + sum_k w_{t,k} Wd_e h_{t,k}
//
// Few tokens go to moe_few.cu (bound by reading the weights, latency), more to moe_tc.cu (tensor cores); this file has the
// routing, the plans that sort (token, place) pairs by expert for either, and the weighted sum behind the latter.
#include <algorithm>
#include <cooperative_groups.h>

#include "moe.cuh"
#include "moe_route.cuh"

namespace cg = cooperative_groups;

namespace mmp {
namespace {

// ------------------------------------------------------------------------------------------------ routing
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
// Exclusive scan of one int2 a thread over a block of 1024 threads.
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

// The plan of the few-token kernels in one block of 1024 threads: groups of at most `G` rows of one expert. V > 0: the
// block routes first (a warp a token), else the expert ids are given.
template <int V, bool F32>
__global__ void __launch_bounds__(1024) moe_plan_few(const MoeArgs A, const RouteParams P, int G) {
  __shared__ int cnt[MOE_MAX_EXPERTS];
  __shared__ int2 warp_tot[32];
  __shared__ short s_e[MOE_FEW_PLACES], s_rank[MOE_FEW_PLACES];
  if constexpr (V == 0) pdl_wait();
  pdl_trigger();  // the next kernel may start; it waits for this one's end before it reads the plan
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int R = A.T * A.places;
  for (int e = tid; e < A.E; e += 1024) cnt[e] = 0;
  if constexpr (V > 0) {
    for (int t = warp; t < A.T; t += 32) {
      int id;
      float w;
      route_token<V, F32>(P, t, lane, id, w);
      if (lane < A.places) {
        P.weights[t * A.places + lane] = w;
        P.ids[t * A.places + lane] = id;
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
  // thread i has expert E - 1 - i: the last expert, which every token may share, comes first
  const int e = A.E - 1 - tid, n = e >= 0 ? cnt[e] : 0, ng = (n + G - 1) / G;
  int2 total;
  const int first = scan_block(make_int2(ng, 0), warp_tot, total).x;
  for (int b = 0; b < ng; ++b) {
    A.groups[first + b].e = e;
    A.groups[first + b].n = min(G, n - b * G);
  }
  if (tid == 0) A.header->ngroups = total.x;
  if (e >= 0) cnt[e] = first;  // this thread alone read the count
  __syncthreads();
  for (int p = tid; p < R; p += 1024) {
    const int q = s_e[p];
    if (q >= 0) A.groups[cnt[q] + s_rank[p] / G].place[s_rank[p] % G] = p;
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
  const int nb = (n + A.block_rows - 1) / A.block_rows;
  int2 total;
  const int2 pre = scan_block(make_int2(n, nb), warp_tot, total);
  const int off = pre.x;
  if (me == 0) {
    for (int b = 0; b < nb; ++b) A.blocks[pre.y + b] = make_int4(e, off, n, b);
    if (tid == 0) A.header->nblk = total.y;
  }
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

// ------------------------------------------------------------------------------------------------ weighted sum
// out_t = addend_t + sum_k w_{t,k} y[pos_{t,k}]: block (token), eight columns a thread.
__global__ void __launch_bounds__(256) moe_combine(const MoeArgs A) {
  pdl_wait();
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
  static int go(const MoeArgs& A, const RouteParams& P, int G, cudaStream_t s) {
    moe_plan_few<V, F32><<<1, 1024, 0, s>>>(A, P, G);
    return mmp_check_launch("mmp_moe_layer");
  }
};

constexpr int FUSED_ROUTE_TOKENS = 32;  // a warp of the planning block a token; more are routed by a launch over the GPU

// The few-token kernels; P.logits set: routing from the logits, else the ids are given.
int few_products(const MoeArgs& A, const RouteParams& P, bool f32, cudaStream_t s) {
  const MoeFewPlan plan = moe_few_plan(A);
  if (plan.tiny) return moe_products_few(A, P, f32, plan, s);
  int rc = MMP_OK;
  if (P.logits && A.T <= FUSED_ROUTE_TOKENS) {
    rc = by_width<LaunchPlan>(P.E, f32, A, P, plan.rows, s);
  } else {
    if (P.logits) rc = by_width<LaunchRoute>(P.E, f32, P, s);
    if (rc != MMP_OK) return rc;
    cudaError_t e = launch_kind(1, moe_plan_few<0, false>, dim3(1), dim3(1024), 0, s, nullptr, 0, A, P, plan.rows);
    if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  }
  return rc != MMP_OK ? rc : moe_products_few(A, P, f32, plan, s);
}

int many_products(MoeArgs& A, const MoeLayout& L, cudaStream_t s) {
  A.block_rows = moe_block_rows(A.T, A.places, A.E);
  cudaError_t e = launch_kind(1, moe_plan_many, dim3(PLAN_BLOCKS), dim3(1024), 0, s, nullptr, 0, A);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  if (!moe_gathers(A.block_rows)) {
    e = launch_kind(1, moe_sort_rows, dim3(A.T), dim3(256), 0, s, nullptr, 0, A);
    if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  }
  const int rc = moe_products_tc(A, L.max_blocks, s);
  if (rc != MMP_OK) return rc;
  e = launch_kind(1, moe_combine, dim3(A.T), dim3(256), 0, s, nullptr, 0, A);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
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
  A.groups = reinterpret_cast<MoeGroup*>(w + L.groups);
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

extern "C" int mmp_moe_launches(int T, int places, int H, int I, int E, int route) {
  if (T <= 0 || places <= 0 || H <= 0 || I <= 0 || E <= 0) return 0;
  if (!moe_is_few(T, places, H, I))  // plan, sorted rows, up, down, sum; routing
    return (moe_gathers(moe_block_rows(T, places, E)) ? 4 : 5) + (route ? 1 : 0);
  MoeArgs A{};
  A.T = T;
  A.places = places;
  A.E = E;
  if (moe_few_plan(A).tiny) return 1;
  return 3 + (route && T > FUSED_ROUTE_TOKENS ? 1 : 0);  // plan (with the routing of few tokens), up, down
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
  return moe_is_few(T, places, H, I) ? few_products(A, RouteParams{}, false, s) : many_products(A, L, s);
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
  if (moe_is_few(T, places, H, I)) return few_products(A, P, logits_dtype == MMP_F32, s);
  rc = by_width<LaunchRoute>(routed, logits_dtype == MMP_F32, P, s);
  return rc != MMP_OK ? rc : many_products(A, L, s);
}
