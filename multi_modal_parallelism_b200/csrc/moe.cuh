// Shared by the mixture-of-experts kernels: the plan that sorts (token, place) pairs by expert, and the workspace it and
// the intermediate rows live in.
//
// A "place" is one (token, slot) pair, numbered t * places + k. The plan lists the places by expert: expert e owns sorted
// rows [off, off + n), sorted row r belongs to place rows[r]. The order of places inside an expert is whatever the
// counting gave: every row is computed by itself, so no result depends on it.
#pragma once
#include <algorithm>

#include "mmp_common.cuh"

namespace mmp {

constexpr int MOE_MAX_EXPERTS = 1024;  // experts in the weight tensors (one thread each in the scan)
constexpr int MOE_MAX_TOPK = 32;       // one lane each in the router
constexpr int MOE_FEW_PLACES = 1152;   // the few-token kernels keep 16 fp32 a place in shared memory (72 KB)
constexpr int MOE_TINY_TOKENS = 8, MOE_TINY_PLACES = 64;  // up to which every block of the few-token kernels plans for itself
// Sorted rows of one expert that the tensor-core kernels take at a time (MMA N): 256, or 128 with a deeper ring of weights
// where experts have few rows.
constexpr int MOE_BLOCK_ROWS = 256, MOE_BLOCK_ROWS_FEW = 128;
// Blocks of 128 rows leave room for a longer ring of weights and let them leave L2 at once (us, 128 / 256 rows a block: 60
// experts, I 1408, 32 rows each 170 / 187, 96 206 / 214, 192 295 / 278; 128 experts, I 768, 48 rows 221 / 231, 128 304 / 293).
inline int moe_block_rows(int64_t T, int places, int E) { return T * places <= 96 * E ? MOE_BLOCK_ROWS_FEW : MOE_BLOCK_ROWS; }
// The up product's kernel of blocks of this many rows gathers them from x; else a kernel before it sorts x (us, gathered /
// sorted: 60 experts, I 1408, 52 rows each 175 / 180; 8 of 176 MB, 8 rows 224 / 231; 256 of 6.3 MB, 64 rows 326 / 337; with 256
// rows the gathers, 16 a block for 64 rows of K, are too many: 2 of 8 large experts, 4096 tokens 1250 / 1094).
__host__ __device__ constexpr bool moe_gathers(int block_rows) { return block_rows == MOE_BLOCK_ROWS_FEW; }

struct MoeHeader {
  int ngroups;  // groups of the few-token kernels
  int nblk;     // row blocks of the tensor-core kernels
  int pad[2];
};

// Few-token kernels: at most 16 places that one expert serves together.
struct MoeGroup {
  int e, n, pad[2];
  int place[16];
};

// Which kernels take a call. Up to 8 tokens and 64 places one launch; then the few-token kernels while the second product is small (R places
// of I columns: its K dimension is I, at which the tensor-core kernels pay 128 columns and an accumulator's turn for each
// expert), the tensor-core kernels else. Measured (us, few-token / tensor-core), H 2048 if not said:
//   257 experts, I 64:  288 places 35 / 64, 1152 71 / 86;   I 128: 576 places 75 / 85, 1152 100 / 99
//   60 experts,  I 256: 128 places 36 / 44, 256 46 / 48, 512 66 / 50;   I 1408: 36 places 91 / 81, 256 192 / 154
//   16 experts,  I 448: 128 places 28 / 30, 256 35 / 31;   257 experts, I 512: 81 places 80 / 82, 288 172 / 158, 576 216 / 206
//   8 experts,   I 2048: 18 places 46 / 46, 64 52 / 46
// The down product of the few-token kernels has a block for 16 columns of H, with few of them it does not fill the GPU:
//   256 experts, H 1024, I 128: 128 places 27 / 35, 256 45 / 42;   I 512: 72 places 66 / 47
// and with many it has two blocks an SM, beside which the results of more places do not fit:
//   64 experts, H 7168, I 64: 512 places 65 / 89, 1024 145 / 96
constexpr int MOE_WIDE = 16 * 148;
inline bool moe_is_tiny(int64_t T, int places) { return T <= MOE_TINY_TOKENS && T * places <= MOE_TINY_PLACES; }
inline bool moe_is_few(int64_t T, int places, int H, int I) {
  const int64_t R = T * places, w = std::min(H, 2048);
  return moe_is_tiny(T, places) || (R <= (H <= MOE_WIDE ? MOE_FEW_PLACES : MOE_FEW_PLACES / 2) && I <= 512 && R * I <= w * w / 64);
}

// Workspace offsets in bytes, every part 256-byte aligned.
struct MoeLayout {
  size_t header, groups, blocks, rows, pos, weights, ids, xs, h, y, bytes;
  int max_blocks;
};

// L2 policy of data that is read once: the first to leave.
__device__ __forceinline__ uint64_t evict_first_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;\n" : "=l"(p));
  return p;
}

inline size_t moe_align(size_t n) { return (n + 255) / 256 * 256; }

inline MoeLayout moe_layout(int64_t T, int places, int H, int I, int E) {
  MoeLayout L;
  const int64_t R = T * places;
  const bool few = moe_is_few(T, places, H, I);
  // the sum over experts of ceil(n / b) is at most R / b + E, and R
  L.max_blocks = static_cast<int>(std::min<int64_t>(R, R / MOE_BLOCK_ROWS_FEW + E));
  size_t at = 0;
  auto part = [&](size_t n) { const size_t o = at; at += moe_align(n); return o; };
  L.header = part(sizeof(MoeHeader));
  const int64_t r = std::min<int64_t>(R, MOE_FEW_PLACES);  // there for more places too: a larger request's scratch serves a smaller one
  L.groups = part(std::min<size_t>(r, r / 8 + E) * sizeof(MoeGroup));
  L.blocks = part(few ? 0 : static_cast<size_t>(L.max_blocks) * 16);
  L.rows = part(few ? 0 : R * 4);
  L.pos = part(few ? 0 : R * 4);
  L.weights = part(R * 4);
  L.ids = part(R * 4);
  L.xs = part(few || moe_gathers(moe_block_rows(T, places, E)) ? 0 : R * H * 2);
  L.h = part(R * I * 2);
  L.y = part(few ? 0 : R * H * 4);
  L.bytes = at;
  return L;
}

// What the kernels get of one call. Strides in elements.
struct MoeArgs {
  const bf16* x; int64_t x_t;
  const bf16* w_gu; int64_t gu_e, gu_r;
  const bf16* w_d; int64_t d_e, d_r;
  const float* weights; int64_t w_t;
  const int32_t* ids; int64_t id_t;
  const bf16* addend; int64_t a_t;
  bf16* out; int64_t o_t;
  int T, places, H, I, E;
  int block_rows;  // tensor-core path
  MoeHeader* header;
  MoeGroup* groups;
  int4* blocks;   // {expert, its first sorted row, its rows, index among its blocks} of the row blocks
  int* rows;      // sorted row -> place
  int* pos;       // place -> sorted row, -1 where the place has no expert
  bf16* xs;       // [sorted row][H]: x in the order of the rows, where they are not gathered
  bf16* h;        // [sorted row][I]; few-token kernels: [place][I]
  float* y;       // [sorted row][H]
  int* err;
};

struct RouteParams {
  const void* logits; int64_t l_t;
  int T, E, top_k, renorm, shared;
  float* weights; int32_t* ids;  // [T, top_k + shared], contiguous
};

// How the few-token kernels take a call: tiny (every block plans for itself, and routes where there are logits), rows of a
// group: 16 where few experts have many rows (us, 8 / 16: 16 experts, H 2048, I 128, 256 places 19.4 / 16.5; 8 experts, H 4096,
// I 256, 64 places 24.6 / 17.2), 8 else (60 experts, H 2048, I 128, 512 places 32 / 39; 64, H 7168, I 128, 512 places 97 / 139).
struct MoeFewPlan { bool tiny; int rows; };
inline MoeFewPlan moe_few_plan(const MoeArgs& A) {
  const bool tiny = moe_is_tiny(A.T, A.places);
  return {tiny, tiny || A.E > 32 || A.T * A.places <= 4 * A.E ? 8 : 16};
}
// The few-token products (moe_few.cu) and the sum into A.out.
int moe_products_few(const MoeArgs& A, const RouteParams& P, bool f32, const MoeFewPlan& plan, cudaStream_t s);

// The tensor-core path (moe_tc.cu): gate/up and down products of a planned call into A.h and A.y.
int moe_products_tc(const MoeArgs& A, int max_blocks, cudaStream_t s);

}  // namespace mmp
