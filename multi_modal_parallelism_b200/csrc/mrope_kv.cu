// Rotary positions with several axes (time, height, width) on q and k, the key multiplier and the paged KV-cache write in
// one pass over the QKV projection. Pair i of the rd / 2 rotated pairs (dims i and i + rd / 2; dims from rd on pass) turns by
//   angle = positions[axes[i], t] * inv_freq[i].
//
// The product is taken as a sum of two doubles and reduced by whole turns (2 pi in two parts, after Cody and Waite) before
// sincosf: in fp32 the angle of position 10^6 would be off by up to 0.03, in fp64 alone that of 10^10 by 1.3e-6, of 10^12 by
// 1.3e-4. One block a token: rd / 2 threads fill the token's cos/sin table once for all its heads (the single-axis kernel
// computes them for every head), then every thread moves 16 + 16 bytes of a rotated head, or 16 of a passing or value part, at
// a time. Bound by HBM (each value is read once and written once): 403 MB for 16384 tokens of 48 heads x 128 in 69 us, 5.8 TB/s.
#include "mmp_common.cuh"

namespace mmp {
namespace {

struct MropeParams {
  const bf16* qkv; int64_t row;
  int nq, nkv, hd, half, naxes;
  const int64_t* positions; int64_t p_a;  // [naxes, T], contiguous rows
  const float* inv_freq;                  // [half]
  const int32_t* axes;                    // [half]
  float key_mult;
  bf16* q_out; int64_t qo_b;
  bf16* kc; bf16* vc; int64_t c_block, c_tok, c_head;
  int block_size, num_blocks;
  const int64_t* slot_mapping;
  int* err;
  uint32_t m_per, m_vper;  // divisors of the task numbering
};

__device__ __forceinline__ float2 turn(int64_t pos, float freq) {
  // 2 pi rounded to fp64 and what that leaves of it, 1 / (2 pi)
  constexpr double TAU = 6.283185307179586476925, TAU_REST = 2.4492935982947064e-16, TURNS = 0.15915494309189533577;
  const double p = static_cast<double>(pos), f = static_cast<double>(freq);  // exact below 2^53
  const double a = p * f, rest = fma(p, f, -a), k = rint(a * TURNS);
  float s, c;
  sincosf(static_cast<float>(fma(-k, TAU_REST, fma(-k, TAU, a) + rest)), &s, &c);
  return make_float2(c, s);
}

__device__ __forceinline__ void unpack8(const uint4& u, float* f) {
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
}
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// n / d by a multiplication with m = ceil(2^32 / d), exact while n * d < 2^32; d == 1: m == 0.
__device__ __forceinline__ int div_by(int n, uint32_t m) { return m ? static_cast<int>(__umulhi(n, m)) : n; }

// W values at a time: 8 (16-byte accesses) where half, hd and every row allow it, else 1.
template <int W>
__global__ void __launch_bounds__(256) mrope_kv_kernel(const MropeParams P) {
  // (cos, sin) of pair i at [i % W][i / W]: neighbouring lanes take neighbouring tasks, so that a read has no bank conflict
  extern __shared__ float2 cs[];
  const int64_t t = blockIdx.x;
  for (int i = threadIdx.x; i < P.half; i += blockDim.x) {
    int a = P.axes[i];
    if (a < 0 || a >= P.naxes) {
      flag_error(P.err, DEVERR_INDEX);
      a = 0;
    }
    cs[i % W * (P.half / W) + i / W] = turn(P.positions[a * P.p_a + t], P.inv_freq[i]);
  }
  const int64_t slot = P.slot_mapping[t];
  int64_t cache = -1;  // this token's offset in the caches, -1: not cached
  if (slot >= 0) {
    const int64_t blk = slot / P.block_size;
    if (blk < P.num_blocks) cache = blk * P.c_block + (slot - blk * P.block_size) * P.c_tok;
    else if (threadIdx.x == 0) flag_error(P.err, DEVERR_INDEX);
  }
  __syncthreads();
  const bf16* src = P.qkv + t * P.row;
  const int rot = P.half / W, per = (P.hd - P.half) / W, vper = P.hd / W;  // tasks: rotated, of a q or k head, of a v head
  const int heads = P.nq + P.nkv, nrot = heads * per, n = nrot + P.nkv * vper;
  for (int q = threadIdx.x; q < n; q += blockDim.x) {
    const bool is_v = q >= nrot;
    const int h = is_v ? div_by(q - nrot, P.m_vper) : div_by(q, P.m_per), j = is_v ? q - nrot - h * vper : q - h * per;
    const bool is_q = !is_v && h < P.nq, pair = !is_v && j < rot;
    const int kvh = is_v ? h : h - P.nq;
    if (!is_q && cache < 0) continue;
    const int d = pair || is_v ? j * W : P.half + j * W;  // first value of the task in its head
    const bf16* s = src + static_cast<int64_t>(is_v ? heads + h : h) * P.hd + d;
    bf16* o = is_q ? P.q_out + t * P.qo_b + static_cast<int64_t>(h) * P.hd + d
                   : (is_v ? P.vc : P.kc) + cache + kvh * P.c_head + d;
    const float mult = is_q || is_v ? 1.f : P.key_mult;
    float lo[W], hi[W];
    if constexpr (W == 8) {
      unpack8(ld16(s), lo);
      if (pair) unpack8(ld16(s + P.half), hi);
    } else {
      lo[0] = bf2f(s[0]);
      if (pair) hi[0] = bf2f(s[P.half]);
    }
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float a = lo[k] * mult;
      lo[k] = a;
      if (pair) {
        const float2 r = cs[k * rot + j];
        const float b = hi[k] * mult;
        lo[k] = a * r.x - b * r.y;
        hi[k] = b * r.x + a * r.y;
      }
    }
    if constexpr (W == 8) {
      st16(o, pack8(lo));
      if (pair) st16(o + P.half, pack8(hi));
    } else {
      o[0] = f2bf(lo[0]);
      if (pair) o[P.half] = f2bf(hi[0]);
    }
  }
}

template <int W>
int launch_mrope(MropeParams P, int T, cudaStream_t s) {
  auto mult = [](int d) { return d > 1 ? static_cast<uint32_t>(((1ull << 32) + d - 1) / d) : 0u; };
  P.m_per = mult((P.hd - P.half) / W);
  P.m_vper = mult(P.hd / W);
  // small blocks where there are enough of them: fewer threads wait for a token's angles (16384 tokens of 48 heads x 128: 69 us
  // with 128 threads, 77 with 256; 64 tokens of 20 heads 3.9 and 3.2)
  mrope_kv_kernel<W><<<T, T < 1024 ? 256 : 128, P.half * sizeof(float2), s>>>(P);
  return mmp_check_launch("mmp_mrope_kv_write");
}

}  // namespace
}  // namespace mmp

using namespace mmp;

extern "C" int mmp_mrope_kv_write(const void* qkv, int64_t row, int nq, int nkv, int hd, const int64_t* positions, int64_t p_a,
                                  int naxes, const float* inv_freq, const int32_t* axes, int rd, float key_mult, void* q_out,
                                  int64_t qo_b, void* key_cache, void* value_cache, int64_t c_block, int64_t c_tok,
                                  int64_t c_head, int block_size, int num_blocks, const int64_t* slot_mapping, int T,
                                  int* err, void* stream) {
  if (T < 0 || nq < 1 || nkv < 1 || hd < 2 || hd > 1024 || rd < 2 || rd > hd || rd % 2 || naxes < 1 || nq > 1024 || nkv > 512 ||
      block_size < 1 || num_blocks < 1)
    return mmp_set_error(MMP_ERR_INVALID, "mmp_mrope_kv_write: T=%d, %d + 2 x %d heads of %d, %d rotated, %d axes, block %d: sizes "
                         "must be positive, hd at most 1024, nq at most 1024 and nkv at most 512, the rotated part even and at most hd", T, nq, nkv, hd, rd, naxes, block_size);
  if (T == 0) return MMP_OK;
  if (!qkv || !positions || !inv_freq || !axes || !q_out || !key_cache || !value_cache || !slot_mapping)
    return mmp_set_error(MMP_ERR_INVALID, "mmp_mrope_kv_write: null pointer");
  if ((T > 1 && (row < static_cast<int64_t>(nq + 2 * nkv) * hd || qo_b < static_cast<int64_t>(nq) * hd)) || p_a < 0)
    return mmp_set_error(MMP_ERR_INVALID, "mmp_mrope_kv_write: rows overlap");
  MropeParams P{static_cast<const bf16*>(qkv), row, nq, nkv, hd, rd / 2, naxes, positions, p_a, inv_freq, axes, key_mult,
                static_cast<bf16*>(q_out), qo_b, static_cast<bf16*>(key_cache), static_cast<bf16*>(value_cache),
                c_block, c_tok, c_head, block_size, num_blocks, slot_mapping, err};
  const bool wide = hd % 8 == 0 && (rd / 2) % 8 == 0 && row % 8 == 0 && qo_b % 8 == 0 && c_block % 8 == 0 && c_tok % 8 == 0 &&
                    c_head % 8 == 0 && aligned16(qkv) && aligned16(q_out) && aligned16(key_cache) && aligned16(value_cache);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return wide ? launch_mrope<8>(P, T, s) : launch_mrope<1>(P, T, s);
}
