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
// Which pair, tile (the longest first) and part a workgroup works on.  Where all are alike: as `share` has it, pair after pair.  Where some tiles are longer (causal): tile after tile over all
// pairs, so that a launch begins with the longest tiles of every pair and not of the first few.  4 x 12 x 1024 x 64: forward 71 us and so 55, dK and dV 107 and 78; 8 x 16 x 2048 x 64, whose
// pairs' keys are four times an XCD's L2 by then: 405 and 340, 696 and 576.  Pairs that do not come in eights go over the XCDs as they come, and their parts one after the other (2 x 14 x
// 1491 x 64: 84 and 65, 129 and 99).  Either side of the border, forward and all gradients, n pairs of 1024 x 64 and of 2048 x 64 pair after pair and tile after tile: 4: 97 and 97, 157 and
// 156 us; 6: 110 and 110, 199 and 180; 9: 142 and 128, 257 and 240; 12: 148 and 140, 285 and 296; 15: 153 and 158, 289 and 297; 24: 167 and 184, 380 and 298; 32: 173 and 174, 466 and 353 (fp32, 4
// pairs of 1024 x 32: 91 and 108).
__host__ __device__ constexpr bool by_tile(int64_t pairs) { return pairs % 8 == 0 || pairs > 8; }
struct dealt {
	uint32_t pair, tile, split;
	__device__ __forceinline__ dealt(uint32_t i, uint32_t pairs, uint32_t tiles, uint32_t splits, bool causal) {
		const bool  eights = (pairs & 7u) == 0u, row_first = causal && by_tile(pairs);
		const share whole(i, pairs, tiles * splits);
		// (eights: a pair on one XCD)
		const uint32_t across = eights ? pairs >> 3 : pairs, j = eights ? i >> 3 : i, row = j / across, turn = j - row * across;
		const uint32_t piece = row_first ? row : whole.piece, in_row = causal && eights ? splits : tiles, outer = piece / in_row, inner = piece - outer * in_row;
		pair  = __builtin_amdgcn_readfirstlane(row_first ? (eights ? 8u * turn + (((i & 7u) - turn) & 7u) : turn) : whole.pair);
		tile  = __builtin_amdgcn_readfirstlane(causal && eights ? outer : inner);
		split = __builtin_amdgcn_readfirstlane(causal && eights ? inner : outer);
	}
};
// ---- rows on their way ----
// The kernels take rows that are whole 16-byte pieces, no further apart than 32 bits reach over a tile; the host lays others out anew (diff_pack_kernel).  With the other way of reading
// beside it in the same loop, as cross_tiles.hpp's passage has it, dK/dV held 756 branches and twice its scalars in vector registers' lanes, and took four times as long.
inline bool takes(int64_t columns, int64_t stride, int bytes) { return columns * bytes % 16 == 0 && stride * bytes < AF3_DIFF_ATTENTION_GRAD_ROW_BYTES; }   // (tiles of 128 rows at most)
// ROWS rows into a tile in LDS, spread over NT threads in 16-byte pieces: one load per piece, at a scalar base and an offset that stays the same from tile to tile
template <typename T, int DP, int ROWS, int NT>
struct carrier {
	using TL = tile<T, DP>;
	static constexpr int N = ROWS * TL::CHUNKS / NT, E = kind<T>::E;
	static_assert(N * NT == ROWS * TL::CHUNKS);
	u32x4    piece[N];
	uint32_t offset[N];   // bytes from the tile's first row
	int64_t  step;        // bytes of a row
	int      D;
	static __device__ __forceinline__ int row_of(int n) { return (threadIdx.x + NT * n) / TL::CHUNKS; }
	static __device__ __forceinline__ int col_of(int n) { return (threadIdx.x + NT * n) % TL::CHUNKS; }
	__device__ __forceinline__ void begin(int64_t stride, int columns) {
		step = stride * (int)sizeof(T), D = columns;
#pragma unroll
		for(int n = 0; n < N; n++) offset[n] = col_of(n) * E < D ? (uint32_t)(row_of(n) * (int)step + col_of(n) * 16) : 0u;
	}
	// rows row0 .. row0 + ROWS - 1 from `base` on, those below `rows` exist (one at least); `like`: one that began with the same strides (this one need not have)
	__device__ __forceinline__ void load(const T* base, int64_t row0, int64_t rows, const carrier& like) {
		const unsigned char* const at   = reinterpret_cast<const unsigned char*>(base) + row0 * like.step;
		const int                  left = rows - row0 < ROWS ? (int)(rows - row0) : ROWS;
#pragma unroll
		for(int n = 0; n < N; n++) piece[n] = load16(reinterpret_cast<const T*>(at + (row_of(n) < left ? like.offset[n] : 0u)));
	}
	__device__ __forceinline__ void load(const T* base, int64_t row0, int64_t rows) { load(base, row0, rows, *this); }
	// all: every row of the tile is wanted; otherwise keep(row) says which, the others become zeros
	template <typename F>
	__device__ __forceinline__ void store(unsigned char* lds, bool all, F keep) const { store(lds, all, keep, D); }
	template <typename F>
	__device__ __forceinline__ void store(unsigned char* lds, bool all, F keep, int columns) const {
#pragma unroll
		for(int n = 0; n < N; n++) {
			u32x4 v = piece[n];
			if(!all || TL::CHUNKS * E != columns) {
				const bool in = (all || keep(row_of(n))) && col_of(n) * E < columns;
#pragma unroll
				for(int i = 0; i < 4; i++) {
					const uint32_t x = v[i];
					v[i] = in ? x : 0u;
				}
			}
			*reinterpret_cast<u32x4*>(lds + row_of(n) * TL::STRIDE + TL::place(row_of(n), col_of(n))) = v;
		}
	}
};
// a row as a B operand in registers, zeros where `ok` is not
template <typename T, int DP, int N>
__device__ __forceinline__ void load_rows(u32x4 (&f)[N], const T* row, bool ok, int columns, int lane) {
	constexpr int E = kind<T>::E;
	static_assert(N == tile<T, DP>::STEPS);
#pragma unroll
	for(int s = 0; s < N; s++) {
		const int d = 2 * E * s + E * (lane >> 5);
		f[s] = u32x4{0u, 0u, 0u, 0u};
		if(ok && d < columns) f[s] = load16(row + d);
	}
}

// 16 results side by side, from column d on, those below D
template <typename T>
__device__ __forceinline__ void store_columns(T* row, int d, int D, const float (&v)[16]) {
	constexpr int E = kind<T>::E;
	if(D % E == 0) {
#pragma unroll
		for(int i = 0; i < 16 / E; i++)
			if(d + E * i < D) store16(row + d + E * i, kind<T>::pack(v + E * i));
	} else {
		store_row16(row, d, D, v);
	}
}

// A reader whose places are worked out again where it is used.  (The exclusive ors of them, 30 to 50 registers, otherwise wait in front of the loop, and operands go to memory instead.)
template <typename R>
__device__ __forceinline__ R fresh(R at) {
	asm volatile("" : "+v"(at.row), "+v"(at.col));
	return at;
}
// the registers of a block whose key (16 half + r from the block's first one on) lies behind the lane's last key become `gone`; `left`: last key - block's first key - 16 half
__device__ __forceinline__ void drop_later(float (&x)[16], int left, float gone) {
#pragma unroll
	for(int r = 0; r < 16; r++) x[r] = r <= left ? x[r] : gone;
}

__device__ __forceinline__ int clamped(int64_t x) { return x > 64 ? 64 : x < -64 ? -64 : (int)x; }

}  // namespace diff

namespace diff {
int width(const af3_diff_attention_params& p);   // columns of a map's queries and keys that a kernel has, half of those of its values

// Up to four tensors [n0, n1, n2, columns] laid out anew where the kernels do not take them as they are: contiguous, rows of whole pieces with zeros at their ends.
struct packing {
	struct job {
		const void* from;
		void*       to;
		int64_t     stride[3], n[3], pieces;
		int32_t     columns;
	} jobs[4];
	int32_t count = 0, element;   // bytes of one
	int64_t bytes = 0;            // of all their places
	explicit packing(int element_) : element(element_) {}
	// `t` and `stride`, where it is not taken as it is, become those of its place in `space` (null: only its size counts); the columns that the kernels see
	int32_t add(const void*& t, int64_t (&stride)[3], int64_t n0, int64_t n1, int64_t n2, int64_t columns, void* space) {
		if(takes(columns, n2 > 1 ? stride[2] : 0, element)) return (int32_t)columns;
		const int64_t whole = (columns * element + 15) / 16 * 16 / element;
		job& j = jobs[count++];
		j = job{t, static_cast<unsigned char*>(space) + bytes, {stride[0], stride[1], stride[2]}, {n0, n1, n2}, n0 * n1 * n2 * whole * element / 16, (int32_t)columns};
		bytes += n0 * n1 * n2 * whole * element;
		t = j.to, stride[0] = n1 * n2 * whole, stride[1] = n2 * whole, stride[2] = whole;
		return (int32_t)whole;
	}
	int launch(hipStream_t s) const;   // (diff_attention.hip)
};
// q, k and v as the kernels take them, in `space` (null: only the sizes count), and the columns of their rows
packing pack_inputs(af3_diff_attention_params& p, int32_t& columns, int32_t& v_columns, void* space);
int64_t packed_bytes(af3_diff_attention_params p);
}  // namespace diff

bool diff_gradients_fit(const af3_diff_attention_params& p);
int  validate_diff_attention(const af3_diff_attention_params* p);

}  // namespace af3
