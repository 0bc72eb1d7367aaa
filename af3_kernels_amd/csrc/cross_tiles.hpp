// What the kernels of attention to states of another length share (cross_attention.hip, cross_attention_grad.hip): tiles of rows in
// LDS, and matrix fragments of them for bf16 and fp32 alike.
//
// Every fragment is 16 bytes per lane, E = 16 / sizeof(T) elements, and one step contracts 2E of them: bf16 one
// v_mfma_f32_32x32x16_bf16, fp32 four v_mfma_f32_32x32x2_f32.  A contraction takes its elements in any order as long as both operands
// do, and so do the 32 rows of a result as long as the reader knows them.  Both freedoms are used the same way everywhere: row i of
// an A operand is tile row tile_row(i), chosen so that register r of a lane in half h of the wavefront holds result row 16 h + r.
// A result's registers, packed, are then the B operand of the next product as they stand (contraction step j: rows 16 h + E j ...),
// a lane's 16 values of a bias row lie side by side in memory, and so do the 16 it stores of a result row.
#pragma once
#include "mfma_helpers.hpp"

namespace af3 {
namespace cross {

constexpr int THREADS = 256, WAVES = 4;
constexpr float LOWEST = -3.402823466e38f;
constexpr float LARGE  = 65536.f;   // of a lane's sum of 16 probabilities: the reference is left behind

template <typename T>
struct kind;
template <>
struct kind<uint16_t> {   // bf16 bits
	static constexpr int E = 8;
	static __device__ __forceinline__ f32x16 mma(const u32x4& a, const u32x4& b, f32x16 c) {
		return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
	}
	// registers E j .. E j + E - 1 of a result as step j of a B operand (rounded to bf16: the product that follows takes nothing wider)
	static __device__ __forceinline__ u32x4 pack(const float* r) { return u32x4{pack_bf16x2(r[0], r[1]), pack_bf16x2(r[2], r[3]), pack_bf16x2(r[4], r[5]), pack_bf16x2(r[6], r[7])}; }
	static __device__ __forceinline__ float at(const u32x4& v, int i) { return i & 1 ? __uint_as_float(v[i >> 1] & 0xffff0000u) : __uint_as_float(v[i >> 1] << 16); }
	static __device__ __forceinline__ float value(uint16_t x) { return bf16_bits_to_f32(x); }
	static __device__ __forceinline__ uint16_t bits(float f) { return (uint16_t)f32_to_bf16_bits(f); }
};
template <>
struct kind<float> {
	static constexpr int E = 4;
	static __device__ __forceinline__ f32x16 mma(const u32x4& a, const u32x4& b, f32x16 c) {
#pragma unroll
		for(int i = 0; i < 4; i++) {
			const uint32_t x = a[i], y = b[i];
			c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x), __uint_as_float(y), c, 0, 0, 0);
		}
		return c;
	}
	static __device__ __forceinline__ u32x4 pack(const float* r) { return u32x4{__float_as_uint(r[0]), __float_as_uint(r[1]), __float_as_uint(r[2]), __float_as_uint(r[3])}; }
	static __device__ __forceinline__ float at(const u32x4& v, int i) {
		const uint32_t x = v[i];
		return __uint_as_float(x);
	}
	static __device__ __forceinline__ float value(float x) { return x; }
	static __device__ __forceinline__ float bits(float f) { return f; }
};

typedef __attribute__((ext_vector_type(4), aligned(4))) uint32_t u32x4_f32;
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p) {   // 16 bytes at any element's address
	if constexpr(sizeof(T) == 2) return *reinterpret_cast<const u32x4_any*>(p);
	else return *reinterpret_cast<const u32x4_f32*>(p);
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const u32x4& v) {
	if constexpr(sizeof(T) == 2) *reinterpret_cast<u32x4_any*>(p) = v;
	else *reinterpret_cast<u32x4_f32*>(p) = v;
}
// E elements of a row from element d on, zeros from D on
template <typename T>
__device__ __forceinline__ u32x4 load_guarded(const T* row, int d, int D) {
	constexpr int E = kind<T>::E;
	T             e[E];
#pragma unroll
	for(int i = 0; i < E; i++) {
		e[i] = T(0);
		if(d + i < D) e[i] = row[d + i];
	}
	return *reinterpret_cast<const u32x4*>(e);
}

__device__ __forceinline__ int   tile_row(int i) { return 16 * ((i >> 2) & 1) + (i & 3) + 4 * (i >> 3); }
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }   // (NaN stays)
// What is taken off a row's logits in units of log2 e, its reference, is a row's maximum (or what was its maximum) times the factor, rounded: every probability of the row is off by the
// same 2^-24 of it.  Far from zero that is felt, and from 2^24 on it alone decides whether they are zero or infinite (rows whose every key has a bias of -1e9, say): such
// rows have their maximum taken off in the logits' own units, where logits near it lose nothing.  Infinite references and NaN are far as well.
constexpr float FAR = 4096.f;
__device__ __forceinline__ bool is_far(float reference) { return !(__builtin_fabsf(reference) < FAR); }
// What the gradients take off a row's logits instead (bf16): the reference and the logarithm of the row's sum together, so that P comes out of the exponential as it is.
// (fp32 keeps the two apart: in one number their rounding, 2^-24 of it, would be the largest error of P.)  1 / sum == 0, a row without a live key, makes P zero.
__device__ __forceinline__ float whole_reference(float m, float inv, float to_log2) { return m * to_log2 - __builtin_amdgcn_logf(inv); }
// a value of lane l and that of lane l ^ 32, joined
__device__ __forceinline__ float sum_of_halves(float x) {
	const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
	return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float maximum_of_halves(float x) {
	const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
	return maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// A tile in LDS: rows of DP elements, whose 16-byte pieces change places by the row so that neither way of reading meets one of the 64 banks twice.  Sixteen lanes
// of a row_frag read rows 0-7 and 16-23 (or 8 more each) at one column: sixteen rows that differ in their bits 0, 1, 2 and 4.  32 lanes of a col_frag of bf16
// read 64 bytes of four consecutive rows, which differ in bits 0 and 1.  So bits 0 and 1 move a piece by 64 bytes and more and bits 2 and 4 within 64 bytes, where
// the rows' own beginnings do not do so already.  (fp32 reads 128 bytes of two rows 16 apart: there bit 4 moves by 128.)  With rows of 16 bytes more instead
// conflicts were 50 of 101 million clocks of LDS work at 8 x 16 x 1491 x 4096 x 128.
template <typename T, int DP>
struct tile {
	static constexpr int STRIDE = DP * (int)sizeof(T), STEPS = DP * (int)sizeof(T) / 32, BLOCKS = DP / 32, CHUNKS = DP * (int)sizeof(T) / 16, JOINTS = 32 / (2 * kind<T>::E);
	// where piece `chunk` of a row lies: 16 (chunk ^ turn(row)), in a part of a row that begins at a multiple of SPAN
	static constexpr int SPAN = STRIDE % 256 == 0 ? 256 : STRIDE % 128 == 0 ? 128 : 64;
	static constexpr __device__ __forceinline__ int turn(int row) {
		const int b0 = row & 1, b1 = (row >> 1) & 1, b2 = (row >> 2) & 1, b4 = (row >> 4) & 1;
		return SPAN == 256 ? (sizeof(T) == 2 ? 8 * b0 | 4 * b1 | 2 * b4 | b2 : 8 * b4 | 4 * b0 | 2 * b1 | b2) : SPAN == 128 ? 4 * b1 | 2 * b4 | b2 : 2 * b4 | b2;
	}
	static __device__ __forceinline__ int place(int row, int chunk) { return 16 * (chunk ^ turn(row)); }
	// Two numbers per lane that all its reads begin with: a read's own place is an exclusive or and a constant away.
	struct reader {
		int row, col;
		__device__ __forceinline__ explicit reader(int lane) {
			const int r = tile_row(lane & 31), half = lane >> 5;
			row = r * STRIDE + place(r, half);
			if constexpr(sizeof(T) == 2) {
				// (ds_read_b64_tr_b16: lane i of a group of 16 supplies 4 columns of row i / 4 and receives 4 rows of the group's column i)
				const int i = lane & 15, G = lane >> 4, c = 16 * (G >> 1) + (i >> 2);
				col = c * STRIDE + place(c, 2 * (i & 1) + (G & 1)) + 8 * ((i >> 1) & 1);
			} else {
				col = 16 * half * STRIDE + place(16 * half, r >> 2) + 4 * (r & 3);
			}
		}
	};
	// contraction over the columns: A operand, step s, of the 32 rows from `row0` (a multiple of 32) on
	static __device__ __forceinline__ u32x4 row_frag(const unsigned char* lds, int row0, int s, const reader& at) {
		return *reinterpret_cast<const u32x4*>(lds + row0 * STRIDE + (at.row ^ (32 * s & (SPAN - 1))) + (32 * s & ~(SPAN - 1)));
	}
	// contraction over the 32 rows from `row0` on: A operand, step j, of columns 32 db .. 32 db + 31
	static __device__ __forceinline__ u32x4 col_frag(const unsigned char* lds, int row0, int db, int j, const reader& at) {
		constexpr int W = 32 * (int)sizeof(T);
		u32x4         f;
		if constexpr(sizeof(T) == 2) {
#pragma unroll
			for(int t = 0; t < 2; t++) {
				const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + row0 * STRIDE + (8 * j + 4 * t) * STRIDE + (at.col ^ ((W * db & (SPAN - 1)) | 16 * turn(4 * t))) + (W * db & ~(SPAN - 1)))));
				f[2 * t] = r[0], f[2 * t + 1] = r[1];
			}
		} else {
#pragma unroll
			for(int t = 0; t < 4; t++) f[t] = *reinterpret_cast<const uint32_t*>(lds + row0 * STRIDE + (4 * j + t) * STRIDE + (at.col ^ ((W * db & (SPAN - 1)) ^ 16 * turn(4 * j + t))) + (W * db & ~(SPAN - 1)));
		}
		return f;
	}
};

// ROWS rows on their way from memory into a tile, spread over the workgroup's threads in 16-byte pieces.  The plain way (rows all there, D a whole number of pieces,
// 32-bit offsets within the tile) is one load per piece at a scalar base and an offset that stays the same from tile to tile.
template <typename T, int DP, int ROWS>
struct passage {
	using TL = tile<T, DP>;
	static constexpr int N = ROWS * TL::CHUNKS / THREADS, E = kind<T>::E;
	static_assert(N * THREADS == ROWS * TL::CHUNKS);
	u32x4    piece[N];
	uint32_t offset[N];   // bytes from the tile's first row
	const T* base;
	int64_t  stride;
	int      D;
	bool     plain;
	static __device__ __forceinline__ int row_of(int n) { return (threadIdx.x + THREADS * n) / TL::CHUNKS; }
	static __device__ __forceinline__ int col_of(int n) { return (threadIdx.x + THREADS * n) % TL::CHUNKS; }
	__device__ __forceinline__ void begin(const T* base_, int64_t stride_, int D_, bool whole) {
		base = base_, stride = stride_, D = D_;
		plain = whole && stride_ <= (int64_t)0x7fffffff / ((int64_t)ROWS * (int)sizeof(T));
#pragma unroll
		for(int n = 0; n < N; n++) offset[n] = plain && col_of(n) * E < D ? (uint32_t)((row_of(n) * (int)stride + col_of(n) * E) * (int)sizeof(T)) : 0u;
	}
	// rows row0 .. row0 + ROWS - 1, those below `rows` exist (one at least)
	__device__ __forceinline__ void load(int64_t row0, int64_t rows) {
		const T*  at   = base + row0 * stride;
		const int left = rows - row0 < ROWS ? (int)(rows - row0) : ROWS;
		if(plain) {
#pragma unroll
			for(int n = 0; n < N; n++) piece[n] = load16(reinterpret_cast<const T*>(reinterpret_cast<const unsigned char*>(at) + (row_of(n) < left ? offset[n] : 0u)));
		} else {
#pragma unroll
			for(int n = 0; n < N; n++) piece[n] = load_guarded(at + (int64_t)(row_of(n) < left ? row_of(n) : 0) * stride, col_of(n) * E, D);
		}
	}
	// all: every row of the tile is wanted; otherwise keep(row) says which, the others become zeros
	template <typename F>
	__device__ __forceinline__ void store(unsigned char* lds, bool all, F keep) const {
#pragma unroll
		for(int n = 0; n < N; n++) {
			u32x4 v = piece[n];
			if(!all || TL::CHUNKS * E != D) {
				const bool in = (all || keep(row_of(n))) && col_of(n) * E < D;
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

// 32 rows of a matrix as a B operand, held in registers: lane holds column (= row of memory) `row`, zeros where `ok` is not
template <typename T, int DP, int N>
__device__ __forceinline__ void load_operand(u32x4 (&f)[N], const T* row, bool ok, int D, int lane) {
	constexpr int E = kind<T>::E;
	static_assert(N == tile<T, DP>::STEPS);
#pragma unroll
	for(int s = 0; s < N; s++) {
		const int d = 2 * E * s + E * (lane >> 5);
		f[s] = u32x4{0u, 0u, 0u, 0u};
		if(ok && d + E <= D) f[s] = load16(row + d);
		else if(ok && d < D) f[s] = load_guarded(row, d, D);
	}
}

// 16 entries of a row from `first` on, those from L on 0 (`row` is the row's first entry)
template <typename T, int N>
__device__ __forceinline__ void load_row16_raw(u32x4 (&out)[N], const T* row, int64_t first, int64_t L) {
	constexpr int E = kind<T>::E;
	static_assert(N == 16 / E);
	if(first + 16 <= L) {
#pragma unroll
		for(int i = 0; i < N; i++) out[i] = load16(row + first + E * i);
	} else {
#pragma unroll
		for(int i = 0; i < N; i++) out[i] = first + E * i < L ? load_guarded(row + first + E * i, 0, L - first - E * i < E ? (int)(L - first - E * i) : E) : u32x4{0u, 0u, 0u, 0u};
	}
}
// 16 results side by side, from element d on, those below D
template <typename T>
__device__ __forceinline__ void store_row16(T* row, int d, int D, const float (&v)[16]) {
	constexpr int E = kind<T>::E;
	if(d + 16 <= D) {
#pragma unroll
		for(int i = 0; i < 16 / E; i++) store16(row + d + E * i, kind<T>::pack(v + E * i));
	} else {
#pragma unroll
		for(int i = 0; i < 16; i++)
			if(d + i < D) row[d + i] = kind<T>::bits(v[i]);
	}
}

// ---- which keys are live ----
// A stretch of SEGMENT keys at a time: one bit per key in `bits`, one bit per tile of KT keys that has a live one in `tiles`.
constexpr int SEGMENT = 16384;
template <int KT>
struct live_keys {
	uint32_t bits[SEGMENT / 32];
	uint32_t tiles[SEGMENT / KT / 32];
	// keys first .. last - 1 (at most SEGMENT of them); a barrier stands before and behind it
	template <int NT = THREADS>
	__device__ __forceinline__ void scan(const uint8_t* mask, int64_t first, int64_t last) {
		__syncthreads();
		for(int i = threadIdx.x; i < SEGMENT / KT / 32; i += NT) tiles[i] = 0u;
		__syncthreads();
		const int n = (int)(last - first);
		for(int k = 32 * threadIdx.x; k < n; k += 32 * NT) {
			uint32_t w = 0u;
			if(!mask) {
				w = n - k >= 32 ? ~0u : (1u << (n - k)) - 1u;
			} else if(n - k >= 32) {
				const u32_bytes* m = reinterpret_cast<const u32_bytes*>(mask + first + k);
#pragma unroll
				for(int i = 0; i < 8; i++) w |= ((live_bytes(m[i]) * 0x01020408u) >> 24) << (4 * i);
			} else {
				for(int i = 0; i < n - k; i++) w |= (mask[first + k + i] != 0 ? 1u : 0u) << i;
			}
			bits[k >> 5] = w;
			if(w) atomicOr(&tiles[(k / KT) >> 5], 1u << ((k / KT) & 31));
		}
		// (the words of a tile that begins below n and ends behind it)
		for(int k = (n + 31) / 32 + threadIdx.x; k < (n + KT - 1) / KT * (KT / 32); k += NT) bits[k] = 0u;
		__syncthreads();
	}
	// the first live tile from t on, -1: none
	__device__ __forceinline__ int next(int t) const {
		for(int w = t >> 5; w < SEGMENT / KT / 32; w++) {
			uint32_t x = tiles[w];
			if(w == t >> 5) x &= ~0u << (t & 31);
			x = (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
			if(x) return 32 * w + __builtin_ctz(x);
		}
		return -1;
	}
};
// the bits of a tile's keys, the same for all lanes
template <int KT>
struct tile_bits {
	static constexpr int N = KT / 32;
	uint32_t word[N];
	__device__ __forceinline__ tile_bits(const live_keys<KT>& live, int t) {
#pragma unroll
		for(int i = 0; i < N; i++) word[i] = (uint32_t)__builtin_amdgcn_readfirstlane((int)live.bits[t * N + i]);
	}
	__device__ __forceinline__ bool full() const {
		uint32_t x = ~0u;
#pragma unroll
		for(int i = 0; i < N; i++) x &= word[i];
		return x == ~0u;
	}
	__device__ __forceinline__ uint32_t of_block(int block) const {
		uint32_t x = word[0];
#pragma unroll
		for(int i = 1; i < N; i++) x = block == i ? word[i] : x;
		return x;
	}
	__device__ __forceinline__ bool keeps(int key) const { return (of_block(key >> 5) >> (key & 31)) & 1u; }   // (a key of the tile, any lane's)
};

// Wavefronts per SIMD that a kernel is to leave room for: three where its accumulators and operands (`registers`) are few, two, or one
constexpr int wavefronts(int registers) { return registers <= 64 ? 3 : registers <= 136 ? 2 : 1; }

// The registers of a block of keys whose bit in `keep` is 0 become `gone`.  (Register r is key r in the lower half-wave, 16 + r in the upper: the lanes that keep theirs
// are a scalar, and one vector instruction per register is left.)
__device__ __forceinline__ void drop_keys(float (&x)[16], uint32_t keep, float gone) {
#pragma unroll
	for(int r = 0; r < 16; r++) {
		const uint64_t lanes = (uint64_t)(uint32_t)((int32_t)(keep << (31 - r)) >> 31) | (uint64_t)(uint32_t)((int32_t)(keep << (15 - r)) >> 31) << 32;
		x[r] = __builtin_amdgcn_inverse_ballot_w64(lanes) ? x[r] : gone;
	}
}

// Into how many parts the long axis of a launch goes: `workgroups` of them walk `tiles` tiles each, `tile_us` apiece, and `slots` fit the chip at a time; a part more
// costs its results' way through memory (`part_bytes`, out and in again) and the kernel that joins them.  The parts of the smallest sum, of two tiles at least.
inline uint32_t parts_for(int64_t workgroups, int64_t slots, int64_t tiles, double tile_us, double part_bytes, int64_t most) {
	constexpr double JOIN_US = 6.0, BYTES_PER_US = 2e6;   // (measured: 6 us with its launch; 2 TB/s)
	double   best = 0.0;
	uint32_t parts = 1;
	for(int64_t n = 1; n <= most && (n == 1 || (2 * n <= tiles + 1 && workgroups * n <= slots)); n++) {
		const double us = (double)((tiles + n - 1) / n) * tile_us + (n > 1 ? JOIN_US + n * 2.0 * part_bytes / BYTES_PER_US : 0.0);
		if(n == 1 || us < best) best = us, parts = (uint32_t)n;
	}
	return parts;
}

// Which (batch, key head) a workgroup works on, and which of its `each` pieces.  Workgroup i runs on XCD i % 8, whose L2 the pieces of one pair share; a pair goes to an XCD
// whole where the pairs divide evenly, and consecutive eights of pairs are turned against each other, so that batch rows of few keys and of many are
// dealt out evenly too (by stretches of consecutive pairs, 8 batch rows of 0.5 to 1 of 1024 keys each had their own XCD: a third of the chip idle).
struct share {
	uint32_t pair, piece;
	__device__ __forceinline__ share(uint32_t i, uint32_t pairs, uint32_t each) {
		if((pairs & 7u) == 0u) {
			const uint32_t xcd = i & 7u, turn = (i >> 3) / each;
			piece = (i >> 3) - turn * each, pair = 8u * turn + ((xcd - turn) & 7u);
		} else {
			const uint32_t n = pairs * each, whole = n & ~7u, k = i < whole ? (i & 7u) * (whole >> 3) + (i >> 3) : i;
			pair = k / each, piece = k - pair * each;
		}
	}
};

}  // namespace cross
}  // namespace af3
