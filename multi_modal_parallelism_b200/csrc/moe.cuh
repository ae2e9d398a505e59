// Shared by the mixture-of-experts kernels: the plan that sorts (token, place) pairs by expert, and the workspace it and
// the intermediate rows live in.
//
// A "place" is one (token, slot) pair, numbered t * places + k. The plan lists the places by expert: expert e owns sorted
// rows [off, off + n), sorted row r belongs to place rows[r]. The order of places inside an expert is whatever the
// counting gave: every row is computed by itself, so no result depends on it.
#pragma once
#include "mmp_common.cuh"

namespace mmp {

constexpr int MOE_MAX_EXPERTS = 1024;  // experts in the weight tensors (one thread each in the scan)
constexpr int MOE_MAX_TOPK = 32;       // one lane each in the router
constexpr int MOE_FEW_PLACES = 1536;   // the few-token kernels keep 16 fp32 a place in shared memory (96 KB)
constexpr int MOE_BLOCK_ROWS = 256;    // sorted rows of one expert that the tensor-core kernels take at a time (MMA N)

struct MoeHeader {
  int nact;  // experts with rows
  int nblk;  // row blocks of the tensor-core kernels
  int pad[2];
};

// Workspace offsets in bytes, every part 256-byte aligned.
struct MoeLayout {
  size_t header, recs, blocks, rows, pos, weights, ids, xs, h, y, bytes;
  int max_blocks;
};

inline size_t moe_align(size_t n) { return (n + 255) / 256 * 256; }

inline MoeLayout moe_layout(int64_t T, int places, int H, int I, int E) {
  MoeLayout L;
  const size_t R = static_cast<size_t>(T) * places;
  const bool few = R <= MOE_FEW_PLACES;
  L.max_blocks = static_cast<int>(R / MOE_BLOCK_ROWS) + E;  // sum over experts of ceil(n / block) is at most this
  size_t at = 0;
  auto part = [&](size_t n) { const size_t o = at; at += moe_align(n); return o; };
  L.header = part(sizeof(MoeHeader));
  L.recs = part(static_cast<size_t>(E) * 16);
  L.blocks = part(static_cast<size_t>(L.max_blocks) * 16);
  L.rows = part(R * 4);
  L.pos = part(R * 4);
  L.weights = part(R * 4);
  L.ids = part(R * 4);
  L.xs = part(few ? 0 : R * H * 2);
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
  MoeHeader* header;
  int4* recs;     // {expert, first sorted row, rows, 0} of the experts with rows, by falling expert
  int4* blocks;   // {expert, its first sorted row, its rows, index among its blocks} of the row blocks
  int* rows;      // sorted row -> place
  int* pos;       // place -> sorted row, -1 where the place has no expert
  bf16* xs;       // [sorted row][H]: x in the order of the rows (tensor-core path)
  bf16* h;        // [sorted row][I]
  float* y;       // [sorted row][H]
  int* err;
};

// The tensor-core path (moe_tc.cu): gate/up and down products of a planned call into A.h and A.y.
int moe_products_tc(const MoeArgs& A, int max_blocks, cudaStream_t s);

}  // namespace mmp
