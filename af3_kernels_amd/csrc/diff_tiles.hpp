// What the kernels of differential attention share (diff_attention.hip, diff_attention_grad.hip), on top of cross_tiles.hpp's tiles and fragments.
//
// Head h of a call is a pair of softmax maps, of query heads 2 h and 2 h + 1 over key heads 2 hk and 2 hk + 1, and one set of values: columns up to DP for queries
// and keys, up to DV = 2 DP for values, results and their gradients.  The G = H / Hkv heads that share a key head are one matrix of G * Lq rows, row R being
// query R / G of head R % G of the group: rows of a tile are then queries side by side, and a causal call leaves out the tiles behind the last of them.
#pragma once
#include "cross_tiles.hpp"

namespace af3 {
namespace diff {

using namespace cross;

// key `j` counts for query `i` of a causal call if j <= i + q_offset
struct row_place {
	int64_t g, qi, h;   // head of the group, query, head of the call
	bool    ok;
	__device__ __forceinline__ row_place(int64_t R, int64_t rows, int64_t G, int64_t hk) {
		ok = R < rows;
		qi = ok ? R / G : 0, g = ok ? R - qi * G : 0, h = hk * G + g;
	}
};
__device__ __forceinline__ float lam_of(const af3_diff_attention_params& p, int64_t h) {
	return p.lam_dtype == AF3_F32 ? static_cast<const float*>(p.lam)[h * p.lam_stride] : bf16_bits_to_f32(static_cast<const uint16_t*>(p.lam)[h * p.lam_stride]);
}
// the registers of a block whose key (16 half + r from the block's first one on) lies behind the lane's last key become `gone`; `left`: last key - block's first key - 16 half
__device__ __forceinline__ void drop_later(float (&x)[16], int left, float gone) {
#pragma unroll
	for(int r = 0; r < 16; r++) x[r] = r <= left ? x[r] : gone;
}

__device__ __forceinline__ int clamped(int64_t x) { return x > 64 ? 64 : x < -64 ? -64 : (int)x; }

}  // namespace diff

bool diff_gradients_fit(const af3_diff_attention_params& p);
int  validate_diff_attention(const af3_diff_attention_params* p);

}  // namespace af3
