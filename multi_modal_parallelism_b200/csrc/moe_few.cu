// Mixture-of-experts products for few tokens: bound by reading each chosen expert's weights once, and by latency.
//
// Weight rows meet up to 8 tokens at a time in mma.m16n8k16 (16 weight rows x 8 tokens). Every warp streams its own weights
// through a queue of steps in shared memory that only it uses: a step is 64 values of its 16 rows and of its tokens' rows,
// copied 16 bytes a lane (the k dimension permuted the same way in both operands, so that a lane's 16 bytes are its fragments
// of two MMAs and each lane reads back what it copied itself: no barrier, no bank conflict). The queue runs on across units
// of work, so that loads stay in flight through their ends.
//   up:   a unit is 8 columns of h for one group of rows (8 gate + 8 up rows are the 16 MMA rows, one thread ends with both
//         of a pair); the 8 warps of a block split its k dimension and meet in shared memory once a unit;
//   down: a block takes 16 columns of the output for ALL experts, its warps take (group, k range) tasks and leave 16 fp32
//         a place in shared memory; then each token's places are summed in their order: no atomics, no partial results in
//         HBM.
// With at most 8 tokens and 64 places (7 tokens of 9) the layer is one launch.
#include <algorithm>
#include <cooperative_groups.h>

#include "moe.cuh"
#include "moe_route.cuh"

namespace cg = cooperative_groups;

namespace mmp {
namespace {

__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes to shared memory, zeros where !valid. Weights are the first to leave L2 (64 tokens x 8 of 256 experts 222 -> 215 us:
// what the next kernels read stays).
__device__ __forceinline__ void copy_weight(uint32_t dst, const bf16* p, bool valid, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint.L2::128B [%0], [%1], 16, %2, %3;\n"
               ::"r"(dst), "l"(p), "r"(valid ? 16 : 0), "l"(policy) : "memory");
}
__device__ __forceinline__ void copy_row(uint32_t dst, const bf16* p, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(p), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

constexpr int STEP = 64;

// A warp's queue of D steps for MT tiles of 16 weight rows and NF groups of 8 tokens. In a slot: 2 x MT x 2 x 512 bytes of
// weights (half step, tile, 8 rows), then 2 x NF x 512 bytes of token rows, 16 bytes a lane each. Weights pass through shared
// memory once in, once out; with 16 tokens their rows did as much again, so that two tiles share them there.
template <int MT, int NF, int D>
struct Queue {
  static constexpr int SLOT = (4 * MT + 2 * NF) * 512;
  static constexpr int BYTES = D * SLOT;
  uint32_t base;  // this lane's 16 bytes of slot 0
  uint64_t policy = evict_first_policy();
  int put = 0, get = 0;

  // this lane's row of every 8: row + tile * of_tile + (second 8) * of_half, from column k on (zeros past K, and in the 8-row
  // pieces from `pieces` on)
  __device__ __forceinline__ void weights(int slot, const bf16* row, int64_t of_tile, int64_t of_half, int pieces, int k, int K) const {
    const uint32_t s = base + slot * SLOT;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = k + h * 32 < K;
      const bf16* p = row + (in ? k + h * 32 : 0);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bool have = m * 2 + j < pieces;
          copy_weight(s + ((h * MT + m) * 2 + j) * 512, have ? p + m * of_tile + j * of_half : p, in && have, policy);
        }
    }
  }
  __device__ __forceinline__ void rows(int slot, const bf16* const (&xr)[NF], const bool (&have)[NF], int k, int K) const {
    const uint32_t s = base + slot * SLOT + 2048 * MT;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = k + h * 32 < K;
      const int kk = in ? k + h * 32 : 0;
#pragma unroll
      for (int f = 0; f < NF; ++f) copy_row(s + (h * NF + f) * 512, xr[f] + kk, in && have[f]);
    }
  }
  __device__ __forceinline__ void pushed() {
    copy_commit();
    put = put + 1 == D ? 0 : put + 1;
  }
  // acc[m][f] (16 rows x 8 tokens) += the oldest step
  __device__ __forceinline__ void pop(float (&acc)[MT][NF][4]) {
    copy_wait<D - 1>();
    const uint32_t s = base + get * SLOT;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 x[NF];
#pragma unroll
      for (int f = 0; f < NF; ++f) x[f] = lds16(s + 2048 * MT + (h * NF + f) * 512);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint4 a = lds16(s + (h * MT + m) * 1024), b = lds16(s + (h * MT + m) * 1024 + 512);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          mma_16816(acc[m][f], a.x, b.x, a.y, b.y, x[f].x, x[f].y);
          mma_16816(acc[m][f], a.z, b.z, a.w, b.w, x[f].z, x[f].w);
        }
      }
    }
    get = get + 1 == D ? 0 : get + 1;
  }
};

template <int MT, int NF>
__device__ __forceinline__ void clear(float (&acc)[MT][NF][4]) {
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[m][f][c] = 0.f;
}

// ------------------------------------------------------------------------------------------------ plan of a few places
struct TinyGroup {
  int e, n;
  int place[8];
};
struct TinyPlan {
  int id[MOE_TINY_PLACES];
  TinyGroup g[MOE_TINY_PLACES];
  int first[MOE_TINY_PLACES];  // of an expert's first place: its first group
  float w[MOE_TINY_PLACES];
  int warp_n[MOE_TINY_PLACES / 32];
  int ngroups;
};

// At most MOE_TINY_PLACES places, by every block for itself (the same in every block): routed where P.logits is set (a warp
// a token), else from the ids. Place p's rank among its expert's is counted by comparing it with every other.
template <int V, bool F32>
__device__ __forceinline__ void tiny_plan(const MoeArgs& A, const RouteParams& P, TinyPlan& S, bool report) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, R = A.T * A.places;
  if constexpr (V > 0) {
    if (warp < A.T) {
      int id;
      float w;
      route_token<V, F32>(P, warp, lane, id, w);
      if (lane < A.places) {
        S.id[warp * A.places + lane] = id;
        S.w[warp * A.places + lane] = w;
      }
    }
  } else if (tid < R) {
    const int t = tid / A.places, k = tid - t * A.places;
    int e = A.ids[t * A.id_t + k];
    if (e >= A.E && report) flag_error(A.err, DEVERR_INDEX);
    S.id[tid] = e < 0 || e >= A.E ? -1 : e;
    S.w[tid] = A.weights[t * A.w_t + k];
  }
  __syncthreads();
  // place tid's rank among its expert's places, their number, and the first of them
  int e = -1, rank = 0, n = 0, lead = tid;
  if (tid < R) {
    e = S.id[tid];
#pragma unroll 4
    for (int q = 0; q < MOE_TINY_PLACES; q += 4) {
      if (q >= R) break;
      const int4 v = *reinterpret_cast<const int4*>(S.id + q);  // past R: no expert's
      const int o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool same = o[c] == e && q + c < R;
        n += same;
        rank += same && q + c < tid;
        if (same) lead = min(lead, q + c);
      }
    }
  }
  // the first place of every expert opens its groups
  const int ng = e >= 0 && rank == 0 ? (n + 7) / 8 : 0;
  int s = ng;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += v;
  }
  if (tid < MOE_TINY_PLACES && lane == 31) S.warp_n[warp] = s;
  __syncthreads();
  int first = s - ng;
  for (int q = 0; q < MOE_TINY_PLACES / 32; ++q)
    if (q < warp) first += S.warp_n[q];
  if (ng > 0) {
    S.first[tid] = first;
    for (int b = 0; b < ng; ++b) {
      S.g[first + b].e = e;
      S.g[first + b].n = min(8, n - b * 8);
    }
  }
  if (tid == 0) {
    int total = 0;
    for (int q = 0; q < MOE_TINY_PLACES / 32; ++q) total += S.warp_n[q];
    S.ngroups = total;
  }
  __syncthreads();
  if (e >= 0) S.g[S.first[lead] + (rank >> 3)].place[rank & 7] = tid;
  __syncthreads();
}

__device__ __forceinline__ int plan_load(const TinyGroup*, const int* p) { return *p; }
__device__ __forceinline__ int plan_load(const MoeGroup*, const int* p) { return __ldcg(p); }

// What a warp knows of a group: the expert, and of each 8 tokens this lane's (token lane / 4): whether there is one, its
// place.
template <int NF>
struct Group {
  int e, place[NF];
  bool have[NF];
  template <typename G>
  __device__ __forceinline__ void load(const G* g, int g4) {
    e = plan_load(g, &g->e);
    const int n = plan_load(g, &g->n);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int p = plan_load(g, &g->place[f * 8 + g4]);
      have[f] = f * 8 + g4 < n;
      place[f] = have[f] ? p : 0;  // what is past the last was not written
    }
  }
};

// ------------------------------------------------------------------------------------------------ up
constexpr int UP_WARPS = 8;

// Units u = u0, u0 + stride, ... by a crew of 8 warps: columns 8 MT (u / ngroups) .. of h for group u % ngroups. red:
// 8 * MT * NF * 32 float4 of the crew; sync(): its barrier. Neighbouring units are of different groups: with those of one group
// next to one another, hundreds of blocks read the same token rows at the same time, and L2 serves a line one after the other
// (32 tokens x 4 of 60 experts, I 1408: the kernel took 117 us instead of 98).
template <int MT, int NF, int D, typename G, typename Sync>
__device__ __forceinline__ void up_units(const MoeArgs& A, const G* groups, int ngroups, int u0, int stride, int warp, int lane,
                                         Queue<MT, NF, D>& q, float4* red, Sync sync) {
  const int g4 = lane >> 2, t4 = lane & 3;
  const int units = (A.I + 8 * MT - 1) / (8 * MT), total = ngroups * units, steps = (A.H + STEP - 1) / STEP;
  const int mine = steps > warp ? (steps - warp + UP_WARPS - 1) / UP_WARPS : 0;  // steps warp, warp + 8, ... of a unit

  // the unit whose steps are being requested, and the group of the one after it
  int pu = u0, ps = 0, pieces = 0;
  const bf16 *row = nullptr, *xr[NF];
  bool have[NF];
  Group<NF> next;
  if (pu < total) next.load(groups + pu % ngroups, g4);
  auto open = [&]() {
    const int i0 = pu / ngroups * 8 * MT;
    row = A.w_gu + next.e * A.gu_e + static_cast<int64_t>(i0 + g4) * A.gu_r + t4 * 8;
    pieces = min(MT, (A.I - i0) / 8) * 2;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      xr[f] = A.x + next.place[f] / A.places * A.x_t + t4 * 8;
      have[f] = next.have[f];
    }
    if (pu + stride < total) next.load(groups + (pu + stride) % ngroups, g4);
  };
  if (pu < total) open();
  auto request = [&]() {
    if (pu < total && mine > 0) {
      const int k = (warp + ps * UP_WARPS) * STEP, kl = A.H - t4 * 8;  // this lane's columns start 8 t4 in
      q.weights(q.put, row, 8 * A.gu_r, A.I * A.gu_r, pieces, k, kl);
      q.rows(q.put, xr, have, k, kl);
      if (++ps == mine) {
        ps = 0;
        pu += stride;
        if (pu < total) open();
      }
    }
    q.pushed();
  };
#pragma unroll
  for (int d = 0; d < D; ++d) request();

  int round = 0;
  for (int u = u0; u < total; u += stride, ++round) {
    float acc[MT][NF][4];
    clear(acc);
    for (int s = 0; s < mine; ++s) {
      q.pop(acc);
      request();
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const float* c = acc[m][f];
        red[(warp * MT * NF + m * NF + f) * 32 + lane] = make_float4(c[0], c[1], c[2], c[3]);
      }
    sync();
    const int b = (warp - round) & (UP_WARPS - 1);
    if (b < MT * NF) {  // one warp for each 8 columns and 8 tokens, another one each round
      const int m = b / NF, f = b % NF;
      float4 v = red[b * 32 + lane];
#pragma unroll
      for (int w = 1; w < UP_WARPS; ++w) {
        const float4 o = red[(w * MT * NF + b) * 32 + lane];
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      const auto* gr = groups + u % ngroups;
      const int n = plan_load(gr, &gr->n), i = (u / ngroups * MT + m) * 8 + g4;
      // h is rounded to bf16, the type of the second product's operands: half a step of 2^-8 relative, as the output's own
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = f * 8 + t4 * 2 + c;
        const float gt = c ? v.y : v.x, up = c ? v.w : v.z;
        if (r < n && i < A.I) A.h[static_cast<int64_t>(plan_load(gr, &gr->place[r])) * A.I + i] = f2bf(silu(gt) * up);
      }
    }
    sync();
  }
  copy_wait<0>();
  q.put = q.get = 0;
}

// ------------------------------------------------------------------------------------------------ down
// How many warps share a group's k range: as it makes the longest warp shortest, at most max_splits. Every lane weighs one
// choice (a loop over them by every thread of a block took 5 us).
__device__ __forceinline__ int down_splits(int ngroups, int steps, int warps, int max_splits, int lane) {
  const int sp = lane + 1;
  uint32_t len = 0xffffffu;
  if (sp <= max_splits) len = min(0xfffffeu, static_cast<uint32_t>((ngroups * sp + warps - 1) / warps * ((steps + sp - 1) / sp)));
  return static_cast<int>(__reduce_min_sync(0xffffffffu, len << 8 | sp) & 255u);
}

__device__ __forceinline__ int down_turn(int ngroups, int tile, int tiles) {
  return static_cast<int>(static_cast<int64_t>(ngroups) * tile / tiles);
}

// Output columns r0 .. r0 + 16 MT - 1: the warps' tasks (group, k range) into val [split][place][16 MT]. Blocks start at
// different groups (`turn`), so that they do not all read the same rows of h at once (32 tokens x 4 of 60 experts, I 1408: the
// kernel took 73 us instead of 64). ready() is called by every warp once its first weights are requested, and returns when
// h is written.
template <int MT, int NF, int D, typename G, typename Ready>
__device__ __forceinline__ void down_tasks(const MoeArgs& A, const G* groups, int ngroups, int splits, int r0, int warp, int warps,
                                           int lane, int turn, Queue<MT, NF, D>& q, float* val, Ready ready) {
  const int g4 = lane >> 2, t4 = lane & 3, R = A.T * A.places, steps = (A.I + STEP - 1) / STEP;
  const int per = (steps + splits - 1) / splits, total = ngroups * splits, kl = A.I - t4 * 8;
  int pt = warp, ps = 0, pend = 0;  // the task whose steps are being requested, its next step and the end of its range
  const bf16 *row = nullptr, *xr[NF];
  bool have[NF];
  auto group = [&](int task) {
    const int g = task / splits + turn;
    return groups + (g < ngroups ? g : g - ngroups);
  };
  Group<NF> next;
  if (pt < total) next.load(group(pt), g4);
  const int pieces = min(2 * MT, (A.H - r0) / 8);  // H is a multiple of 8
  auto open = [&]() {
    row = A.w_d + next.e * A.d_e + static_cast<int64_t>(r0 + g4) * A.d_r + t4 * 8;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      xr[f] = A.h + static_cast<int64_t>(next.place[f]) * A.I + t4 * 8;
      have[f] = next.have[f];
    }
    ps = pt % splits * per;
    pend = min(steps, ps + per);
    if (pt + warps < total) next.load(group(pt + warps), g4);
  };
  auto advance = [&]() {  // to the next step; tasks whose range is empty are passed
    ++ps;
    while (ps >= pend && pt < total) {
      pt += warps;
      if (pt < total) open();
    }
  };
  if (pt < total) {
    open();
    if (ps >= pend) advance();
  }
  const int early = pt < total ? min(D, pend - ps) : 0;
  for (int d = 0; d < early; ++d) q.weights(d, row, 16 * A.d_r, 8 * A.d_r, pieces, (ps + d) * STEP, kl);
  ready();
#pragma unroll
  for (int d = 0; d < D; ++d) {
    if (pt < total) {
      if (d >= early) q.weights(d, row, 16 * A.d_r, 8 * A.d_r, pieces, ps * STEP, kl);
      q.rows(d, xr, have, ps * STEP, kl);
      advance();
    }
    q.pushed();
  }
  for (int task = warp; task < total; task += warps) {
    const int sp = task % splits;
    const auto* gr = group(task);
    const int n = plan_load(gr, &gr->n);
    int place[NF][2];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int c = 0; c < 2; ++c) place[f][c] = f * 8 + t4 * 2 + c < n ? plan_load(gr, &gr->place[f * 8 + t4 * 2 + c]) : -1;
    float acc[MT][NF][4];
    clear(acc);
    for (int s = sp * per; s < min(steps, (sp + 1) * per); ++s) {
      q.pop(acc);
      if (pt < total) {
        q.weights(q.put, row, 16 * A.d_r, 8 * A.d_r, pieces, ps * STEP, kl);
        q.rows(q.put, xr, have, ps * STEP, kl);
        advance();
      }
      q.pushed();
    }
    float* v = val + static_cast<int64_t>(sp) * R * 16 * MT + g4;
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (place[f][c] >= 0)
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            v[(place[f][c] * MT + m) * 16] = acc[m][f][c];
            v[(place[f][c] * MT + m) * 16 + 8] = acc[m][f][c + 2];
          }
  }
  copy_wait<0>();
  q.put = q.get = 0;
}

// The addend of this thread's first columns in down_sum, read before the products so that its latency passes meanwhile.
template <int MT>
__device__ __forceinline__ uint32_t down_addend(const MoeArgs& A, int r0) {
  const int t = threadIdx.x / (8 * MT), c = threadIdx.x % (8 * MT) * 2;
  return A.addend && t < A.T && r0 + c < A.H ? *reinterpret_cast<const uint32_t*>(A.addend + t * A.a_t + r0 + c) : 0u;
}

// Each token's places in their order, two columns a thread. have(p): whether place p has an expert, weight(p): its weight.
template <int MT, typename Have, typename Weight>
__device__ __forceinline__ void down_sum(const MoeArgs& A, int splits, int r0, const float* val, uint32_t first, Have have,
                                         Weight weight) {
  const int R = A.T * A.places;
  for (int j = threadIdx.x; j < A.T * 8 * MT; j += blockDim.x) {
    const int t = j / (8 * MT), c = j % (8 * MT) * 2;
    if (r0 + c >= A.H) continue;
    if (j != static_cast<int>(threadIdx.x)) first = A.addend ? *reinterpret_cast<const uint32_t*>(A.addend + t * A.a_t + r0 + c) : 0u;
    float2 s = unpack_bf16x2(first);
#pragma unroll 4
    for (int k = 0; k < A.places; ++k) {
      const int p = t * A.places + k;
      float y0 = 0.f, y1 = 0.f;
      for (int sp = 0; sp < splits; ++sp) {
        const float2 v = *reinterpret_cast<const float2*>(val + (static_cast<int64_t>(sp) * R + p) * 16 * MT + c);
        y0 += v.x;
        y1 += v.y;
      }
      if (have(p)) {  // else nothing was written there
        const float w = weight(p);
        s.x = fmaf(w, y0, s.x);
        s.y = fmaf(w, y1, s.y);
      }
    }
    *reinterpret_cast<uint32_t*>(A.out + t * A.o_t + r0 + c) = pack_bf16x2(s.x, s.y);
  }
}

// ------------------------------------------------------------------------------------------------ planned: two kernels
template <int MT, int NF, int D>
constexpr int up_shared() {
  return UP_WARPS * Queue<MT, NF, D>::BYTES + UP_WARPS * MT * NF * 512;
}

template <int MT, int NF, int D>
__global__ void __launch_bounds__(UP_WARPS * 32, NF == 1 ? 4 : 2) moe_up_few(const MoeArgs A) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Queue<MT, NF, D> q;
  q.base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * Queue<MT, NF, D>::BYTES + lane * 16;
  pdl_wait();
  pdl_trigger();  // after the wait: what was planned is then visible to the next kernel before its own wait
  up_units(A, A.groups, __ldcg(&A.header->ngroups), blockIdx.x, gridDim.x, warp, lane, q,
           reinterpret_cast<float4*>(smem + UP_WARPS * Queue<MT, NF, D>::BYTES), []() { __syncthreads(); });
}

// Shared memory: the queues, the places' results, their weights and whether they have an expert.
template <int WARPS, int MT, int NF, int D>
constexpr int down_shared(int R, int splits) {
  return WARPS * Queue<MT, NF, D>::BYTES + R * (64 * MT * splits + 8);
}

// Block b: output columns 16 MT b .. of every token.
template <int WARPS, int MT, int NF, int D>
__global__ void __launch_bounds__(WARPS * 32) moe_down_few(const MoeArgs A, int max_splits) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int R = A.T * A.places, r0 = blockIdx.x * 16 * MT;
  float* val = reinterpret_cast<float*>(smem + WARPS * Queue<MT, NF, D>::BYTES);  // [split][place][16 MT]
  float* s_w = val + static_cast<int64_t>(max_splits) * R * 16 * MT;
  int* s_ok = reinterpret_cast<int*>(s_w + R);
  // the plan is complete: the kernel before this one let it start only after its own wait for it
  const int ngroups = __ldcg(&A.header->ngroups);
  for (int p = tid; p < R; p += WARPS * 32) {
    const int t = p / A.places, k = p - t * A.places, e = __ldcg(A.ids + t * A.id_t + k);
    s_w[p] = __ldcg(A.weights + t * A.w_t + k);
    s_ok[p] = e >= 0 && e < A.E;
  }
  const int splits = down_splits(ngroups, (A.I + STEP - 1) / STEP, WARPS, max_splits, lane);
  Queue<MT, NF, D> q;
  q.base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * Queue<MT, NF, D>::BYTES + lane * 16;
  uint32_t first = 0;
  down_tasks(A, A.groups, ngroups, splits, r0, warp, WARPS, lane, down_turn(ngroups, blockIdx.x, gridDim.x), q, val, [&]() {
    pdl_wait();
    first = down_addend<MT>(A, r0);
  });
  pdl_trigger();
  __syncthreads();
  down_sum<MT>(A, splits, r0, val, first, [=](int p) { return s_ok[p] != 0; }, [=](int p) { return s_w[p]; });
}

// ------------------------------------------------------------------------------------------------ tiny: one kernel
// At most 8 tokens and 64 places: the whole layer in one cooperative launch of a block an SM. Every block plans (and routes)
// for itself; four crews of 8 warps take up units; then every warp requests its first down weights and the grid meets; then
// all 32 warps take down tasks. 1 token x 9 of 257 experts (H 2048, I 512): 21.4 us, as two launches 24.7.
constexpr int TINY_WARPS = 32, TINY_D = 2, TINY_RED = TINY_WARPS * 512;
constexpr int TINY_SHARED = TINY_WARPS * Queue<1, 1, TINY_D>::BYTES + TINY_RED + static_cast<int>(sizeof(TinyPlan));

template <int V, bool F32>
__global__ void __launch_bounds__(TINY_WARPS * 32, 1) moe_tiny(const MoeArgs A, const RouteParams P) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, crew = warp / UP_WARPS;
  uint8_t* red = smem + TINY_WARPS * Queue<1, 1, TINY_D>::BYTES;  // up: the crews' partial sums; down: the places' results
  TinyPlan& S = *reinterpret_cast<TinyPlan*>(red + TINY_RED);
  Queue<1, 1, TINY_D> q;
  q.base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * Queue<1, 1, TINY_D>::BYTES + lane * 16;
  tiny_plan<V, F32>(A, P, S, blockIdx.x == 0);
  up_units(A, S.g, S.ngroups, blockIdx.x + gridDim.x * crew, gridDim.x * (TINY_WARPS / UP_WARPS), warp % UP_WARPS, lane, q,
           reinterpret_cast<float4*>(red + crew * UP_WARPS * 512),
           [=]() { asm volatile("bar.sync %0, %1;\n" ::"r"(crew + 1), "n"(UP_WARPS * 32) : "memory"); });
  const int R = A.T * A.places, tiles = (A.H + 15) / 16;
  const int splits = down_splits(S.ngroups, (A.I + STEP - 1) / STEP, TINY_WARPS, TINY_RED / (R * 64), lane);
  float* val = reinterpret_cast<float*>(red);
  bool met = false;
  for (int tile = blockIdx.x; tile < tiles || !met; tile += gridDim.x) {
    auto meet = [&]() {
      if (!met) cg::this_grid().sync();
      met = true;
    };
    if (tile >= tiles) {  // a block without columns
      meet();
      break;
    }
    const uint32_t first = down_addend<1>(A, tile * 16);
    down_tasks(A, S.g, S.ngroups, splits, tile * 16, warp, TINY_WARPS, lane, down_turn(S.ngroups, tile, tiles), q, val, meet);
    __syncthreads();
    down_sum<1>(A, splits, tile * 16, val, first, [&](int p) { return S.id[p] >= 0; }, [&](int p) { return S.w[p]; });
    __syncthreads();  // the results are overwritten next
  }
}

// ------------------------------------------------------------------------------------------------ host side
template <typename K>
int allow_shared(K kern, int bytes, bool (&set)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && set[dev]) return MMP_OK;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: shared memory attribute: %s", cudaGetErrorString(e));
  if (dev >= 0 && dev < 64) set[dev] = true;
  return MMP_OK;
}

constexpr int SM_SHARED = 227 * 1024;  // shared memory of an SM for blocks
static_assert(TINY_SHARED <= SM_SHARED, "moe_tiny");

template <int V, bool F32>
int launch_tiny(const MoeArgs& A, const RouteParams& P, int sms, cudaStream_t s) {
  auto kern = moe_tiny<V, F32>;
  static bool set[64] = {};
  int rc = allow_shared(kern, TINY_SHARED, set);
  if (rc != MMP_OK) return rc;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;  // the grid meets once
  attr[0].val.cooperative = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms);
  cfg.blockDim = dim3(TINY_WARPS * 32);
  cfg.dynamicSmemBytes = TINY_SHARED;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, A, P);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  return mmp_check_launch("mmp_moe_experts");
}

template <int MT, int NF>
int launch_up(const MoeArgs& A, int max_groups, int sms, cudaStream_t s) {
  constexpr int D = 2, bytes = up_shared<MT, NF, D>();
  auto kern = moe_up_few<MT, NF, D>;
  static bool set[64] = {};
  int rc = allow_shared(kern, bytes, set);
  if (rc != MMP_OK) return rc;
  constexpr int per_sm = std::min(NF == 1 ? 4 : 2, SM_SHARED / (bytes + 1024));
  const int64_t units = static_cast<int64_t>(max_groups) * ((A.I + 8 * MT - 1) / (8 * MT));
  const int grid = static_cast<int>(std::min<int64_t>(units, static_cast<int64_t>(sms) * per_sm));
  cudaError_t e = launch_kind(1, kern, dim3(grid), dim3(UP_WARPS * 32), bytes, s, nullptr, 0, A);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  return MMP_OK;
}

template <int WARPS, int MT, int NF, int D>
int launch_down(const MoeArgs& A, int limit, cudaStream_t s) {
  auto kern = moe_down_few<WARPS, MT, NF, D>;
  static bool set[64] = {};
  int rc = allow_shared(kern, SM_SHARED, set);
  if (rc != MMP_OK) return rc;
  const int R = A.T * A.places;
  int splits = 1;
  while (splits < WARPS && down_shared<WARPS, MT, NF, D>(R, splits + 1) <= limit) ++splits;
  cudaError_t e = launch_kind(1, kern, dim3((A.H + 16 * MT - 1) / (16 * MT)), dim3(WARPS * 32),
                              down_shared<WARPS, MT, NF, D>(R, splits), s, nullptr, 0, A, splits);
  if (e != cudaSuccess) return mmp_set_error(MMP_ERR_CUDA, "mmp_moe_experts: %s", cudaGetErrorString(e));
  return MMP_OK;
}

// 16 warps while one block an SM covers the columns, else two blocks of 8 while the results fit beside their queues.
static_assert(down_shared<16, 1, 1, 3>(MOE_FEW_PLACES, 1) <= SM_SHARED && down_shared<8, 1, 2, 2>(MOE_FEW_PLACES, 1) <= SM_SHARED,
              "there is a choice for any request");

int products8(const MoeArgs& A, int max_groups, int sms, cudaStream_t s) {
  int rc = launch_up<1, 1>(A, max_groups, sms, s);
  if (rc != MMP_OK) return rc;
  if ((A.H + 15) / 16 <= sms) return launch_down<16, 1, 1, 3>(A, SM_SHARED, s);
  return launch_down<8, 1, 1, 3>(A, std::max(SM_SHARED / 2 - 1024, down_shared<8, 1, 1, 3>(A.T * A.places, 1)), s);
}

int products16(const MoeArgs& A, int max_groups, int sms, cudaStream_t s) {
  int rc = launch_up<2, 2>(A, max_groups, sms, s);
  if (rc != MMP_OK) return rc;
  const int R = A.T * A.places, half = SM_SHARED / 2 - 1024;
  if ((A.H + 31) / 32 <= sms && down_shared<16, 2, 2, 2>(R, 1) <= SM_SHARED) return launch_down<16, 2, 2, 2>(A, SM_SHARED, s);
  if (down_shared<8, 2, 2, 2>(R, 1) <= half) return launch_down<8, 2, 2, 2>(A, half, s);
  return launch_down<8, 1, 2, 2>(A, SM_SHARED, s);
}

}  // namespace

int moe_products_few(const MoeArgs& A, const RouteParams& P, bool f32, const MoeFewPlan& plan, cudaStream_t s) {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (sms <= 0) sms = 148;
  if (plan.tiny) {
    if (!P.logits) return launch_tiny<0, false>(A, P, sms, s);
    if (P.E <= 64) return f32 ? launch_tiny<2, true>(A, P, sms, s) : launch_tiny<2, false>(A, P, sms, s);
    if (P.E <= 256) return f32 ? launch_tiny<8, true>(A, P, sms, s) : launch_tiny<8, false>(A, P, sms, s);
    return f32 ? launch_tiny<32, true>(A, P, sms, s) : launch_tiny<32, false>(A, P, sms, s);
  }
  const int R = A.T * A.places, most = std::min(R, R / plan.rows + A.E);
  const int rc = plan.rows == 8 ? products8(A, most, sms, s) : products16(A, most, sms, s);
  return rc != MMP_OK ? rc : mmp_check_launch("mmp_moe_experts");
}

}  // namespace mmp
