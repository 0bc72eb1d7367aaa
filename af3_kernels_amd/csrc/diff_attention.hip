// Differential attention: out_h = (softmax(scale q1.k1) - lam_h softmax(scale q2.k2)) . v, two maps over one set of values, bf16 or fp32.
// af3_diff_attention_forward.
//
// Per 32 query rows and 32 keys and map:  S^T[key][row] = K . Q^T,  O^T[column][row] += V^T . P^T,  as in cross_attention.hip: a lane holds one query row, the half-waves 16
// keys each.  The two maps are different wavefronts' (both maps' sums of twice D columns would leave one wavefront to a SIMD), which share the tiles of V; each keeps its own
// running maximum and sum, and the difference is taken at the end, since neither sum is known before.
// Bound by its vector and matrix instructions, which take turns, and by waits of wavefronts that share tiles: 2 x 16 (4) x 4096 x 64 causal 284 us, 727 TFLOP/s (a large product of the
// library: 1306); 4 x 8 x 1024 x 128 83 us, 620.  Workgroups of 4 wavefronts, two to a compute unit, gain 7 % where a launch is short (68 us for 73 at 4 x 12 x 1024 x 64 causal, dealt out pair by pair) and
// lose up to 40 % (128 columns).
#include "diff_tiles.hpp"

#include <math.h>

namespace af3 {
namespace diff {

struct forward_args {
	af3_diff_attention_params p;
	uint32_t row_tiles, splits;    // workgroups per (batch, key head); parts of the key axis
	int64_t  part;                 // keys per part, a multiple of the tile
	float    factor;               // exp2((t - max) * factor) with t = q.k
	int32_t  columns, v_columns;   // of q and k, of v, as they are read: whole pieces
	float*   part_out;             // [splits][2][B * Hkv * G * Lq][Dv] and ...
	void*    values;               // V as fp16, tile after tile, and its tiles' units, or null
	float*   units;
	float*   part_stat;            // ... [splits][2][B * Hkv * G * Lq][2] (maximum, sum); sum 0: no live key in the part, and nothing written
};

// eight results side by side, from column d on, those below D
template <typename T>
__device__ __forceinline__ void store_eight(T* row, int d, int D, const float (&v)[8]) {
	constexpr int E = kind<T>::E;
	if(D % E == 0) {
#pragma unroll
		for(int i = 0; i < 8 / E; i++)
			if(d + E * i < D) store16(row + d + E * i, kind<T>::pack(v + E * i));
	} else {
#pragma unroll
		for(int e = 0; e < 8; e++)
			if(d + e < D) row[d + e] = kind<T>::bits(v[e]);
	}
}

// (what a result loses by its rounding to bf16 is left as bf16 itself: the gradient's row sums then have the result to 16 bits)
// one column of a result, and of the second map's own
template <typename T>
__device__ __forceinline__ void store_result(const af3_diff_attention_params& p, int64_t b, int64_t h, int64_t qi, int64_t row, int column, float v, float second) {
	static_cast<T*>(p.out)[b * p.out_stride[0] + h * p.out_stride[1] + qi * p.out_stride[2] + column] = kind<T>::bits(v);
	if(p.second) static_cast<T*>(p.second)[row * p.Dv + column] = kind<T>::bits(second);
	if constexpr(sizeof(T) == 2)
		if(p.residuals) {
			T* const lost = static_cast<T*>(p.residuals) + row * p.Dv + column;
			lost[0] = kind<T>::bits(v - (float)(__bf16)v);
			lost[p.B * p.H * p.Lq * p.Dv] = kind<T>::bits(second - (float)(__bf16)second);
		}
}

// ---- rows of whole pieces ----
__global__ void __launch_bounds__(THREADS) diff_pack_kernel(packing k) {
	int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
	int     which = 0;
	while(which < k.count && i >= k.jobs[which].pieces) i -= k.jobs[which++].pieces;
	if(which == k.count) return;
	const packing::job& j = k.jobs[which];
	const int     each = 16 / k.element, per_row = (j.columns + each - 1) / each;
	const int64_t row = i / per_row, n2 = row % j.n[2], n1 = row / j.n[2] % j.n[1], n0 = row / j.n[2] / j.n[1];
	const int     c0 = (int)(i - row * per_row) * each;
	const int64_t from = n0 * j.stride[0] + n1 * j.stride[1] + n2 * j.stride[2];
	u32x4 v = {0u, 0u, 0u, 0u};
	for(int c = 0; c < each && c0 + c < j.columns; c++) {
		if(k.element == 4) v[c] = static_cast<const uint32_t*>(j.from)[from + c0 + c];
		else v[c >> 1] |= (uint32_t)static_cast<const uint16_t*>(j.from)[from + c0 + c] << (16 * (c & 1));
	}
	static_cast<u32x4*>(j.to)[i] = v;
}
int packing::launch(hipStream_t s) const {
	int64_t pieces = 0;
	for(int i = 0; i < count; i++) pieces += jobs[i].pieces;
	if(pieces == 0) return AF3_OK;
	if(pieces > (int64_t)0xffffff * THREADS) return AF3_ERR_BAD_SHAPE;
	hipLaunchKernelGGL(diff_pack_kernel, dim3((uint32_t)((pieces + THREADS - 1) / THREADS)), dim3(THREADS), 0, s, *this);
	return launch_status();
}

// ---- the values as fp16 ----
// The rounding of P to bf16 in front of its product with V would be felt more here than in one map: where the maps have much in common their difference loses size and
// the roundings do not (lam 0.8, logits of variance 1: out off by 1.6 times its own last rounding).  In short launches, whose matrix instructions are few, P goes in two terms, the second
// what the first one lost.  In long ones it goes as fp16, which has three bits more, and V with it: its bf16 values times a power of two, the tile's unit, are fp16 values as they stand
// (but for the smallest of a tile).  Laid out so once, rows of dropped keys as zeros, a tile is then taken as it is by all that read it.  Converted
// where it is read instead, 2 x 16 (4) x 4096 x 64 took 352 us in place of 278 (between two barriers, with no other workgroup on the compute unit to fill them).
constexpr int   value_rows(int dp) { return dp == 32 ? 128 : 64; }   // (a whole number of the main kernel's tiles)
constexpr float UNIT = 256.f;   // of the sums in front of the first tile, and of tiles of which nothing else is known
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
	const f16x2 p = {(_Float16)lo, (_Float16)hi};
	return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ u32x4 pack_f16(const float* r) { return u32x4{pack_f16x2(r[0], r[1]), pack_f16x2(r[2], r[3]), pack_f16x2(r[4], r[5]), pack_f16x2(r[6], r[7])}; }
__device__ __forceinline__ f32x16 mma_f16(const u32x4& a, const u32x4& b, f32x16 c) {
	return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// A tile's unit takes its largest value to 2^8 .. 2^15: bf16 values of 2^-25 of it and more are then fp16 values without a rounding, smaller ones off by 2^-33 of it at most.  Within that all tiles of
// a pair have the same one, which suits the largest of some values all along the keys: a tile of another unit than the one before it has the sums multiplied (with the nearest unit for each
// tile, 2 x 16 (4) x 4096 x 64 of values of 0.25 took 306 us, so 283).
constexpr float LEAST = 256.f, MOST_UNITS = 32768.f;
// a power of two that takes x to 2^11 .. 2^12 (x of 2^-89 and more; smaller ones, and zero, by 2^100)
__device__ __forceinline__ float unit_for(float x) {
	int e = 11 + 127 - (int)(__float_as_uint(x) >> 23);
	e     = e > 100 ? 100 : e;
	return __uint_as_float((uint32_t)(e + 127) << 23);
}
// a tile of V per workgroup: [pair][rows up to a whole number of tiles][2 DP], columns from Dv on zeros
template <int DP>
__global__ void __launch_bounds__(THREADS) diff_values_kernel(forward_args a) {
	constexpr int VALUE_ROWS = value_rows(DP);
	using P = carrier<uint16_t, 2 * DP, VALUE_ROWS, THREADS>;
	const af3_diff_attention_params& p = a.p;
	__shared__ float largest[2][WAVES];   // of the tile, of the pair's values that are looked at
	const uint32_t tiles = (uint32_t)((p.Lk + VALUE_ROWS - 1) / VALUE_ROWS), pair = blockIdx.x / tiles, tile_no = blockIdx.x - pair * tiles;
	const int64_t  b = pair / (uint32_t)p.Hkv, hk = pair - (uint32_t)b * (uint32_t)p.Hkv, row0 = (int64_t)tile_no * VALUE_ROWS;
	const uint8_t* const mask = p.key_mask ? p.key_mask + b * p.key_mask_stride_b : nullptr;
	const uint16_t* const base = static_cast<const uint16_t*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[1];
	P v;
	v.begin(p.v_stride[2], a.v_columns);
	v.load(base, row0, p.Lk);
	// (a piece of one of THREADS / CHUNKS rows for each thread)
	const int64_t key    = P::row_of(0) * p.Lk / (THREADS / P::TL::CHUNKS);
	const bool    column = P::col_of(0) * P::E < a.v_columns;
	const u32x4   piece  = load16(base + key * p.v_stride[2] + (column ? P::col_of(0) * P::E : 0));
	const bool    looked = column && (!mask || mask[key] != 0);
	auto larger = [](float top, const u32x4& of, bool in) {   // (neither infinities nor NaN, which no unit changes)
#pragma unroll
		for(int e = 0; e < 8; e++) {
			const float x = __builtin_fabsf(kind<uint16_t>::at(of, e));
			if(in && x < INFINITY) top = __builtin_fmaxf(x, top);
		}
		return top;
	};
	float top = 0.f;
	bool  in[P::N];
#pragma unroll
	for(int n = 0; n < P::N; n++) {
		const int row = P::row_of(n);
		in[n] = row0 + row < p.Lk && P::col_of(n) * P::E < a.v_columns && (!mask || mask[row0 + row] != 0);
		top   = larger(top, v.piece[n], in[n]);
	}
	float looked_at = larger(0.f, piece, looked);
#pragma unroll
	for(int d = 32; d; d >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, d)), looked_at = __builtin_fmaxf(looked_at, __shfl_xor(looked_at, d));
	if((threadIdx.x & 63) == 0) largest[0][threadIdx.x >> 6] = top, largest[1][threadIdx.x >> 6] = looked_at;
	__syncthreads();
#pragma unroll
	for(int w = 0; w < WAVES; w++) top = __builtin_fmaxf(top, largest[0][w]), looked_at = __builtin_fmaxf(looked_at, largest[1][w]);
	// (zeros have the largest unit where the values that were looked at are zeros too: it takes nothing away from other tiles)
	const float usual = looked_at == 0.f && top != 0.f ? UNIT : unit_for(looked_at);
	const float unit = top == 0.f || (top * usual >= LEAST && top * usual < MOST_UNITS) ? usual : unit_for(top);
	if(threadIdx.x == 0) a.units[blockIdx.x] = unit;
	u32x4* const out = static_cast<u32x4*>(a.values) + (int64_t)blockIdx.x * VALUE_ROWS * P::TL::CHUNKS;
#pragma unroll
	for(int n = 0; n < P::N; n++) {
		u32x4 h;
#pragma unroll
		for(int i = 0; i < 4; i++) h[i] = in[n] ? pack_f16x2(kind<uint16_t>::at(v.piece[n], 2 * i) * unit, kind<uint16_t>::at(v.piece[n], 2 * i + 1) * unit) : 0u;
		out[threadIdx.x + THREADS * n] = h;
	}
}

// Eight wavefronts: two maps x KW that share 32 query rows and each take 32 keys of a tile (1: a wavefront takes all keys of one) x 4 / KW blocks of 32 rows
constexpr int   NT   = 512;
constexpr float MOST = 32768.f;   // of a lane's sum of 16 probabilities, which fp16 has to hold: the reference is left behind
constexpr int tile_keys(int bytes, int kw) { return kw == 4 || bytes <= 64 ? 128 : kw == 2 || bytes <= 128 ? 64 : 32; }   // bytes of a row of K
template <typename T, int DP, int KW>
struct forward_shape {
	static constexpr int DV = 2 * DP, KT = tile_keys(DP * (int)sizeof(T), KW), SUB = KT / (32 * KW), GROUPS = 4 / KW, ROWS = 32 * GROUPS;
	static constexpr int KTILE = KT * tile<T, DP>::STRIDE, VTILE = KT * tile<T, DV>::STRIDE, SET = 2 * KTILE + VTILE;
	static constexpr int BUFFERS = 2 * SET <= 65536 ? 2 : 1;
	static constexpr int LINE = DV + 4, TABLE = 32 * LINE * 4;   // results of 32 rows on their way to another wavefront
	static constexpr int PASS = 2, RESULT_LINE = 32 * PASS + 4, RESULTS = 2 * GROUPS * 32 * RESULT_LINE * 4;   // both maps' results, 64 columns of them
	static constexpr int JOIN = KW > 1 ? 4 * TABLE : 0, LEAST = JOIN > RESULTS ? JOIN : RESULTS, LDS = BUFFERS * SET > LEAST ? BUFFERS * SET : LEAST;
};

// HALF: V comes as diff_values_kernel has laid it out
template <typename T, int DP, int KW, bool HALF>
__global__ void __launch_bounds__(NT, 2) diff_forward_kernel(forward_args a) {
	using S  = forward_shape<T, DP, KW>;
	using TK = tile<T, DP>;
	using TV = tile<T, S::DV>;
	constexpr int E = kind<T>::E, KT = S::KT, VALUE_ROWS = value_rows(DP);
	static_assert(!HALF || VALUE_ROWS % KT == 0);
	const af3_diff_attention_params& p = a.p;
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ live_keys<KT> live;
	__shared__ float         stat[8][32][2];
	__shared__ int64_t       out_at[S::ROWS], row_at[S::ROWS];   // of the rows: where their results go, -1: no row
	__shared__ float         lam_at[S::ROWS];
	__shared__ bool          any_key[2][S::ROWS];   // of the rows: whether a map has a live key

	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
	const int map = wave & 1, kwave = (wave >> 1) % KW, group = (wave >> 1) / KW;
	const dealt    own((uint32_t)blockIdx.x, (uint32_t)(p.B * p.Hkv), a.row_tiles, a.splits, p.causal != 0);
	const uint32_t split = own.split, row_tile = a.row_tiles - 1 - own.tile;   // (causal: those with the most keys first)
	const int64_t  b = own.pair / (uint32_t)p.Hkv, hk = own.pair - (uint32_t)b * (uint32_t)p.Hkv;
	const int64_t G = p.H / p.Hkv, rows = G * p.Lq;
	const int     Dv = (int)p.Dv;

	const int64_t   R = (int64_t)row_tile * S::ROWS + 32 * group + (lane & 31);
	const row_place at_row(R, rows, G, hk);
	const bool      ok = at_row.ok;
	const int64_t   qi = at_row.qi, h = at_row.h;
	u32x4 qf[TK::STEPS];
	load_rows<T, DP>(qf, static_cast<const T*>(p.q) + b * p.q_stride[0] + (2 * h + map) * p.q_stride[1] + qi * p.q_stride[2], ok, a.columns, lane);
	const T* const kb = static_cast<const T*>(p.k) + b * p.k_stride[0] + 2 * hk * p.k_stride[1];
	const int64_t  v_rows = HALF ? (p.Lk + VALUE_ROWS - 1) / VALUE_ROWS * VALUE_ROWS : 0;
	const T* const vb = HALF ? static_cast<const T*>(a.values) + own.pair * v_rows * S::DV : static_cast<const T*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[1];
	const float* const units = a.units + own.pair * (v_rows / VALUE_ROWS);
	float unit = HALF ? UNIT : 1.f, coming = unit, p_scale = 1.f, least = 0.f;   // of the sums, of the tile on its way; least: the smallest one so far, 0: none
	const uint8_t* const mask = p.key_mask ? p.key_mask + b * p.key_mask_stride_b : nullptr;

	// p = exp2(t * to_log2 - reference), reference = to_log2 * (a maximum of the row's logits so far)
	const float to_log2 = a.factor;
	float  m = LOWEST, reference = -INFINITY, l = 0.f;
	bool   moves = true;   // the reference moves at the next block (the first one, and while a row is far)
	f32x16 o[TV::BLOCKS];
#pragma unroll
	for(int db = 0; db < TV::BLOCKS; db++) o[db] = f32x16{};

	int64_t last = (int64_t)(split + 1) * a.part < p.Lk ? (int64_t)(split + 1) * a.part : p.Lk;
	if(p.causal) {   // (behind the last key of the workgroup's last query nothing counts)
		const int64_t end_row = (int64_t)(row_tile + 1) * S::ROWS < rows ? (int64_t)(row_tile + 1) * S::ROWS : rows, end = (end_row - 1) / G + p.q_offset + 1;
		last = end < last ? end : last;
	}
	const int64_t limit = p.causal ? qi + p.q_offset : (int64_t)1 << 41;   // the lane's last key
	const typename TK::reader at_k_(lane);
	const typename TV::reader at_v_(lane);
	carrier<T, DP, KT, NT>    pk[2];
	carrier<T, S::DV, KT, NT> pv;
	pk[0].begin(p.k_stride[2], a.columns);
	if constexpr(HALF) pv.begin(S::DV, S::DV);
	else pv.begin(p.v_stride[2], a.v_columns);
	int buffer = 0;
	for(int64_t first = (int64_t)split * a.part; first < last; first += SEGMENT) {
		const int64_t end = first + SEGMENT < last ? first + SEGMENT : last;
		live.template scan<NT>(mask, first, end);
		int t = live.next(0);
		if(t < 0) continue;
		const int within = limit - first > SEGMENT ? SEGMENT : limit - first < -1 ? -1 : (int)(limit - first);
		float coming_next = UNIT;
		auto  fetch = [&](int tile_no) {
			const int64_t from = first + (int64_t)tile_no * KT;
			pk[0].load(kb, from, end), pk[1].load(kb + p.k_stride[1], from, end, pk[0]), pv.load(vb, from, HALF ? v_rows : end);
			if constexpr(HALF) coming_next = units[from / VALUE_ROWS];
		};
		fetch(t);
		while(t >= 0) {
			unsigned char*       ks = smem + buffer * S::SET;
			unsigned char* const vs = ks + 2 * S::KTILE;
			const tile_bits<KT> bits(live, t);
			const bool          full = bits.full();
			const int following = live.next(t + 1);
			coming = coming_next;
			if constexpr(S::BUFFERS == 1) __syncthreads();
			// (what K holds at a dropped key stays in that key's logits, which are not looked at; its row of V meets a weight of zero, and must not be NaN)
			pk[0].store(ks, true, [](int) { return true; });
			pk[1].store(ks + S::KTILE, true, [](int) { return true; }, a.columns);
			if constexpr(HALF) pv.store(vs, true, [](int) { return true; });
			else pv.store(vs, full, [&](int row) { return bits.keeps(row); });
			__syncthreads();
			if constexpr(HALF) {
				p_scale = 1.f;
				if(coming != unit) {   // (no more than 2^60 times the smallest one, so that the sums stay finite: what is missing goes to P)
					const float to = least == 0.f ? coming : __builtin_fminf(coming, least * 0x1p60f), by = least == 0.f ? 1.f : to / unit;
					unit = to;
#pragma unroll
					for(int db = 0; db < TV::BLOCKS; db++) o[db] *= by;
					p_scale = unit / coming;
				}
				least   = least == 0.f ? unit : __builtin_fminf(least, unit);
			}
			if(following >= 0) fetch(following);
			ks += map * S::KTILE;
#pragma unroll 1
			for(int s = 0; s < S::SUB; s++) {
				const int      block = kwave * S::SUB + s;
				const uint32_t keep = bits.of_block(block);
				const int      left = within - (t * KT + 32 * block + 16 * half);   // the lane's keys 0 .. left of its 16 count
				if(keep == 0u || !__any(ok && left >= 0)) continue;
				const bool diagonal = __any(ok && left < 15);
				const typename TK::reader at_k = DP * sizeof(T) > 128 ? fresh(at_k_) : at_k_;
				const typename TV::reader at_v = DP * sizeof(T) > 128 ? fresh(at_v_) : at_v_;
				float x[16];
				auto  logits = [&] {
					f32x16 acc{};
#pragma unroll
					for(int st = 0; st < TK::STEPS; st++) acc = kind<T>::mma(TK::row_frag(ks, 32 * block, st, at_k), qf[st], acc);
#pragma unroll
					for(int r = 0; r < 16; r++) x[r] = acc[r];
					if(keep != ~0u) drop_keys(x, keep, -INFINITY);
					if(diagonal) drop_later(x, left, -INFINITY);
				};
				auto probabilities = [&]() -> float {
					float sum = 0.f;
#pragma unroll
					for(int r = 0; r < 16; r++) {
						x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], to_log2, -reference));
						sum += x[r];
					}
					return sum;
				};
				// (optimistic, as in cross_attention.hip: against the reference as it is, which moves where probabilities get large)
				float sum = 0.f;
				logits();
				if(!moves) {
					sum   = probabilities();
					moves = __any(!(sum < MOST));
					if(moves) logits();
				}
				if(moves) {
					float top = x[0];
#pragma unroll
					for(int r = 1; r < 16; r++) top = maximum(top, x[r]);
					const float to = maximum(m, maximum_of_halves(top)), by = __builtin_amdgcn_exp2f((m - to) * to_log2);
					m = to, reference = m * to_log2, l *= by;
#pragma unroll
					for(int db = 0; db < TV::BLOCKS; db++) o[db] *= by;
					moves = __any(is_far(reference));
					if(moves) {
						sum = 0.f;
#pragma unroll
						for(int r = 0; r < 16; r++) {
							x[r] = __builtin_amdgcn_exp2f((x[r] - m) * to_log2);
							sum += x[r];
						}
					} else {
						sum = probabilities();
					}
				}
				l += sum;
				if(HALF && p_scale != 1.f) {
#pragma unroll
					for(int r = 0; r < 16; r++) x[r] *= p_scale;
				}
#pragma unroll
				for(int j = 0; j < TV::JOINTS; j++) {
					u32x4 pf, lo;
					if constexpr(HALF) pf = pack_f16(x + E * j);
					else pf = kind<T>::pack(x + E * j);
					if constexpr(sizeof(T) == 2 && !HALF) {   // (what pf lost)
						float y[E];
#pragma unroll
						for(int e = 0; e < E; e++) y[e] = x[E * j + e] - kind<T>::at(pf, e);
						lo = kind<T>::pack(y);
					}
#pragma unroll
					for(int db = 0; db < TV::BLOCKS; db++) {
						const u32x4 vf = TV::col_frag(vs, 32 * block, db, j, at_v);
						if constexpr(HALF) o[db] = mma_f16(vf, pf, o[db]);
						else o[db] = kind<T>::mma(vf, pf, o[db]);
						if constexpr(sizeof(T) == 2 && !HALF) o[db] = kind<T>::mma(vf, lo, o[db]);
					}
				}
			}
			t = following;
			if constexpr(S::BUFFERS == 2) buffer ^= 1;
		}
	}
	l = sum_of_halves(l);

	float* const tables = reinterpret_cast<float*>(smem);   // four of them, 32 rows each
	const int    line = (lane & 31) * S::LINE + 16 * half;
	auto put = [&](float* table, int db, float by) {
#pragma unroll
		for(int e = 0; e < 4; e++) *reinterpret_cast<f32x4*>(table + line + 32 * db + 4 * e) = f32x4{o[db][4 * e] * by, o[db][4 * e + 1] * by, o[db][4 * e + 2] * by, o[db][4 * e + 3] * by};
	};
	if constexpr(KW > 1) {   // wavefronts that share rows: each weights its own sums by the common maximum, then a part of the columns each; map after map
		if(half == 0) stat[wave][lane][0] = m, stat[wave][lane][1] = l;
		__syncthreads();   // (and nobody reads tiles any more)
		float to = LOWEST, sum = 0.f;
#pragma unroll
		for(int w = 0; w < KW; w++) to = maximum(to, stat[2 * (group * KW + w) + map][lane & 31][0]);
#pragma unroll
		for(int w = 0; w < KW; w++) sum += stat[2 * (group * KW + w) + map][lane & 31][1] * __builtin_amdgcn_exp2f((stat[2 * (group * KW + w) + map][lane & 31][0] - to) * a.factor);
		const float by = __builtin_amdgcn_exp2f((m - to) * a.factor);
		m = to, l = sum;
#pragma unroll
		for(int turn = 0; turn < 2; turn++) {
			if(turn == map) {
#pragma unroll
				for(int db = 0; db < TV::BLOCKS; db++) put(tables + (wave >> 1) * (S::TABLE / 4), db, by);
			}
			__syncthreads();
			if(turn == map) {
#pragma unroll
				for(int db = 0; db < TV::BLOCKS; db++) {
					if(db % KW != kwave) continue;
					o[db] = f32x16{};
#pragma unroll
					for(int w = 0; w < KW; w++)
#pragma unroll
						for(int e = 0; e < 4; e++) {
							const f32x4 v = *reinterpret_cast<const f32x4*>(tables + (group * KW + w) * (S::TABLE / 4) + line + 32 * db + 4 * e);
#pragma unroll
							for(int c = 0; c < 4; c++) o[db][4 * e + c] += v[c];
						}
				}
			}
			__syncthreads();
		}
	}
	const bool  first_of_row = ok && kwave == 0 && half == 0;
	const float per_unit = 1.f / unit;
	if(a.splits > 1) {
		const int64_t n_rows = p.B * p.Hkv * rows, place = (2 * (int64_t)split + map) * n_rows + (b * p.Hkv + hk) * rows + R;
		if(first_of_row) a.part_stat[2 * place] = m, a.part_stat[2 * place + 1] = l;
		if(!ok || l == 0.f) return;
#pragma unroll
		for(int db = 0; db < TV::BLOCKS; db++) {
			if(db % KW != kwave) continue;
			float v[16];
#pragma unroll
			for(int r = 0; r < 16; r++) v[r] = o[db][r] * per_unit;
			store_columns(a.part_out + place * Dv, 32 * db + 16 * half, Dv, v);
		}
		return;
	}
	const float   inv = l == 0.f ? 0.f : 1.f / l, inv_units = inv * per_unit;   // (0: no live key)
	const int64_t row = (b * p.H + h) * p.Lq + qi;
	if(p.stats && first_of_row) {
		float* const st = p.stats + 2 * ((b * 2 * p.H + 2 * h + map) * p.Lq + qi);
		st[0] = m, st[1] = inv;
	}
	// Both maps' results by way of LDS, 64 columns at a time, from where eight of a row are stored in one go and the row by lanes side by side (by the lanes that have them, 16 columns
	// of 32 rows at once, 4 x 12 x 1024 rows over 64 keys with the four results that a gradient needs took 28 us, so 24; 4 x 8 x 1024 x 128 without them 92 and 85).
	if(kwave == 0 && half == 0) any_key[map][32 * group + lane] = l != 0.f;
	if(map == 0 && kwave == 0 && half == 0) {
		const int at = 32 * group + lane;
		out_at[at] = ok ? b * p.out_stride[0] + h * p.out_stride[1] + qi * p.out_stride[2] : -1;
		row_at[at] = row, lam_at[at] = l == 0.f ? 0.f : lam_of(p, h);
	}
	constexpr int PASS = S::PASS, LINE = S::RESULT_LINE, PIECES = 4 * PASS;
	float* const  mine = tables + (2 * group + map) * (32 * LINE) + (lane & 31) * LINE + 16 * half;
#pragma unroll
	for(int first = 0; first < TV::BLOCKS; first += PASS) {
		if(32 * first >= Dv) break;
		__syncthreads();
#pragma unroll
		for(int j = 0; j < PASS; j++) {
			const int db = first + j;
			if(db % KW != kwave) continue;
#pragma unroll
			for(int e = 0; e < 4; e++)
				*reinterpret_cast<f32x4*>(mine + 32 * j + 4 * e) = f32x4{o[db][4 * e] * inv_units, o[db][4 * e + 1] * inv_units, o[db][4 * e + 2] * inv_units, o[db][4 * e + 3] * inv_units};
		}
		__syncthreads();
		for(int n = threadIdx.x; n < S::ROWS * PIECES; n += NT) {
			const int     at = n / PIECES, column = 8 * (n - at * PIECES), d = 32 * first + column;
			const int64_t to = out_at[at], lost_row = row_at[at];
			if(to < 0 || d >= Dv) continue;
			const float* const from = tables + 2 * (at / 32) * (32 * LINE) + (at & 31) * LINE + column;
			const float        lam = lam_at[at];
			const bool         live1 = any_key[0][at], live2 = any_key[1][at];   // (without one: zeros, also where other rows' keys reach the sums with weights of zero, which NaN does not heed)
			float              v[8], second[8];
#pragma unroll
			for(int i = 0; i < 2; i++) {
				const f32x4 one = *reinterpret_cast<const f32x4*>(from + 4 * i), two = *reinterpret_cast<const f32x4*>(from + 32 * LINE + 4 * i);
#pragma unroll
				for(int e = 0; e < 4; e++) second[4 * i + e] = live2 ? two[e] : 0.f, v[4 * i + e] = __builtin_fmaf(-lam, second[4 * i + e], live1 ? one[e] : 0.f);
			}
			store_eight(static_cast<T*>(p.out) + to, d, Dv, v);
			if(!p.second) continue;
			store_eight(static_cast<T*>(p.second) + lost_row * Dv, d, Dv, second);
			if constexpr(sizeof(T) == 2)
				if(p.residuals) {
#pragma unroll
					for(int e = 0; e < 8; e++) v[e] -= (float)(__bf16)v[e], second[e] -= (float)(__bf16)second[e];
					T* const lost = static_cast<T*>(p.residuals) + lost_row * Dv;
					store_eight(lost, d, Dv, v), store_eight(lost + p.B * p.H * p.Lq * Dv, d, Dv, second);
				}
		}
	}
}

// ---- few query rows ----
// Up to 16 rows to a pair of key heads, single tokens above all, are bound by the bytes of K and V and by what a launch costs before them.  The 32 rows of a product are then both maps of
// 16 rows: lanes 0 .. 15 of each half have the first map's, the others the second's; both products of K are taken for all and each lane keeps its own map's logits, so that softmax
// and the product with V are there once.  K comes straight from memory as the products' operand, V by way of LDS of the wavefront's own, 32 keys at a time: wavefronts wait for nobody
// until the end, and 16 KB (D = 64) of each are on their way while it works.  P in two terms.  One token of 32 requests over 1491 keys (16 heads on 4, D = 64): 34.5 us with the kernel
// above, whose 8 wavefronts share tiles, 25.5 with this one; over 8192 keys 143 and 105 (5.1 TB/s).  A step of 128 keys takes 2 us (D = 64; 3 at D = 128) wherever its bytes come in
// time, so a long axis of few requests goes over parts of one step: 8192 keys of one request 27 us in 32 parts of a join that branched, 15 now.
template <typename T, int DP>
struct token_shape {
	static constexpr int DV = 2 * DP, TILE = 32 * tile<T, DV>::STRIDE, AT_ONCE = DV * (int)sizeof(T) / 128, LINE = 32 * AT_ONCE + 4, TABLE = 32 * LINE * 4;   // a tile of V; as many columns of results as have its room: of a wavefront
	static constexpr int LDS = WAVES * (TILE > TABLE ? TILE : TABLE);
};
template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, (DP * sizeof(T) <= 128 ? 2 : 1)) diff_token_kernel(forward_args a) {
	using S  = token_shape<T, DP>;
	using TK = tile<T, DP>;
	using TV = tile<T, S::DV>;
	constexpr int E = kind<T>::E, N = TV::CHUNKS * 32 / 64;   // N: pieces of V per lane
	const af3_diff_attention_params& p = a.p;
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ float stat[WAVES][32][2], inverse[32];

	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, map = (lane >> 4) & 1;
	const share    own((uint32_t)blockIdx.x, (uint32_t)(p.B * p.Hkv), a.splits);
	const uint32_t split = own.piece;
	const int64_t  b = own.pair / (uint32_t)p.Hkv, hk = own.pair - (uint32_t)b * (uint32_t)p.Hkv;
	const int64_t  G = p.H / p.Hkv, rows = G * p.Lq;
	const int      Dv = (int)p.Dv;

	const row_place at_row(lane & 15, rows, G, hk);
	u32x4 qf[TK::STEPS];
	load_rows<T, DP>(qf, static_cast<const T*>(p.q) + b * p.q_stride[0] + (2 * at_row.h + map) * p.q_stride[1] + at_row.qi * p.q_stride[2], at_row.ok, a.columns, lane);
	const T* const kb = static_cast<const T*>(p.k) + b * p.k_stride[0] + 2 * hk * p.k_stride[1];
	const T* const vb = static_cast<const T*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[1];
	const uint8_t* const mask = p.key_mask ? p.key_mask + b * p.key_mask_stride_b : nullptr;
	const float to_log2 = a.factor;
	float  m = LOWEST, reference = -INFINITY, l = 0.f;
	bool   moves = true;
	f32x16 o[TV::BLOCKS];
#pragma unroll
	for(int db = 0; db < TV::BLOCKS; db++) o[db] = f32x16{};

	int64_t last = (int64_t)(split + 1) * a.part < p.Lk ? (int64_t)(split + 1) * a.part : p.Lk;
	if(p.causal) last = p.Lq + p.q_offset < last ? p.Lq + p.q_offset : last;   // (behind the last query's last key nothing counts)
	const int64_t limit = p.causal ? at_row.qi + p.q_offset : (int64_t)1 << 41;   // the lane's last key
	const typename TV::reader at_v(lane);
	unsigned char* const vs = smem + wave * S::TILE;
	const int my_row = tile_row(lane & 31);

	// 32 keys from key0 on: which count at all, and their loads
	auto keys_of = [&](int64_t key0) -> uint32_t {
		const int64_t key = key0 + (lane & 31);
		return (uint32_t)__ballot(key < last && (!mask || mask[key] != 0));
	};
	auto next = [&](int64_t& key0, uint32_t& keep) {   // the first 32 from key0 on that have one that counts (the wavefronts' in turn)
		for(keep = 0u; key0 < last && (keep = keys_of(key0)) == 0u; key0 += 32 * WAVES) {}
	};
	u32x4 kf[2][TK::STEPS], vp[N];
	auto fetch_k = [&](int64_t key0) {
		const int64_t key = key0 + my_row < last ? key0 + my_row : last - 1;
		const T* const row = kb + key * p.k_stride[2];
#pragma unroll
		for(int i = 0; i < 2; i++)
#pragma unroll
			for(int s = 0; s < TK::STEPS; s++) {
				const int d = 2 * E * s + E * half;
				kf[i][s] = u32x4{0u, 0u, 0u, 0u};
				if(d < a.columns) kf[i][s] = load16(row + i * p.k_stride[1] + d);
			}
	};
	auto fetch_v = [&](int64_t key0) {
#pragma unroll
		for(int n = 0; n < N; n++) {
			const int     piece = lane + 64 * n, row = piece / TV::CHUNKS, col = piece % TV::CHUNKS;
			const int64_t key = key0 + row < last ? key0 + row : last - 1;
			vp[n] = u32x4{0u, 0u, 0u, 0u};
			if(col * E < a.v_columns) vp[n] = load16(vb + key * p.v_stride[2] + col * E);
		}
	};
	int64_t  key0 = (int64_t)split * a.part + 32 * wave;
	uint32_t keep;
	next(key0, keep);
	if(keep != 0u) fetch_k(key0), fetch_v(key0);
	while(keep != 0u) {
		int64_t  following = key0 + 32 * WAVES;
		uint32_t keep_following;
		next(following, keep_following);
		f32x16 s1{}, s2{};
#pragma unroll
		for(int s = 0; s < TK::STEPS; s++) s1 = kind<T>::mma(kf[0][s], qf[s], s1), s2 = kind<T>::mma(kf[1][s], qf[s], s2);
		float x[16];
#pragma unroll
		for(int r = 0; r < 16; r++) x[r] = map == 0 ? s1[r] : s2[r];
		if(keep_following != 0u) fetch_k(following);
		if(keep != ~0u) drop_keys(x, keep, -INFINITY);
		if(p.causal) drop_later(x, clamped(limit - key0 - 16 * half), -INFINITY);
		// (a block's own maximum each time: the exponentials are few)
		float top = x[0];
#pragma unroll
		for(int r = 1; r < 16; r++) top = maximum(top, x[r]);
		top = maximum_of_halves(top);
		if(moves || __any(!((top - m) * to_log2 < 14.f))) {
			const float to = maximum(m, top), by = __builtin_amdgcn_exp2f((m - to) * to_log2);
			m = to, reference = m * to_log2, l *= by;
#pragma unroll
			for(int db = 0; db < TV::BLOCKS; db++) o[db] *= by;
			moves = __any(is_far(reference));
		}
		float sum = 0.f;
#pragma unroll
		for(int r = 0; r < 16; r++) {
			x[r] = __builtin_amdgcn_exp2f(moves ? (x[r] - m) * to_log2 : __builtin_fmaf(x[r], to_log2, -reference));
			sum += x[r];
		}
		l += sum;
		// V: what is there by now into LDS (rows that do not count as zeros: theirs are weights of zero, which NaN does not heed), the next one's loads behind it
#pragma unroll
		for(int n = 0; n < N; n++) {
			const int  piece = lane + 64 * n, row = piece / TV::CHUNKS, col = piece % TV::CHUNKS;
			const bool in = ((keep >> row) & 1u) != 0u;
			u32x4      v = vp[n];
#pragma unroll
			for(int i = 0; i < 4; i++) {
				const uint32_t w = v[i];
				v[i] = in ? w : 0u;
			}
			*reinterpret_cast<u32x4*>(vs + row * TV::STRIDE + TV::place(row, col)) = v;
		}
		if(keep_following != 0u) fetch_v(following);
		__builtin_amdgcn_wave_barrier();   // (the wavefront's own LDS: in order)
#pragma unroll
		for(int j = 0; j < TV::JOINTS; j++) {
			const u32x4 pf = kind<T>::pack(x + E * j);
			u32x4       lo;
			if constexpr(sizeof(T) == 2) {   // (what pf lost)
				float y[E];
#pragma unroll
				for(int e = 0; e < E; e++) y[e] = x[E * j + e] - kind<T>::at(pf, e);
				lo = kind<T>::pack(y);
			}
#pragma unroll
			for(int db = 0; db < TV::BLOCKS; db++) {
				const u32x4 vf = TV::col_frag(vs, 0, db, j, at_v);
				o[db] = kind<T>::mma(vf, pf, o[db]);
				if constexpr(sizeof(T) == 2) o[db] = kind<T>::mma(vf, lo, o[db]);
			}
		}
		__builtin_amdgcn_wave_barrier();
		key0 = following, keep = keep_following;
	}
	l = sum_of_halves(l);
	if(half == 0) stat[wave][lane][0] = m, stat[wave][lane][1] = l;
	__syncthreads();   // (and nobody reads a tile any more)
	float to = LOWEST;
#pragma unroll
	for(int w = 0; w < WAVES; w++) to = maximum(to, stat[w][lane & 31][0]);
	const float by = __builtin_amdgcn_exp2f((m - to) * to_log2);
	const int64_t n_rows = p.B * p.Hkv * rows, first_row = (b * p.Hkv + hk) * rows;
	if(threadIdx.x < 32) {   // one of the two maps of a row
		const int       row = threadIdx.x & 15, i = threadIdx.x >> 4;
		const row_place place(row, rows, G, hk);
		float           total = 0.f;
#pragma unroll
		for(int w = 0; w < WAVES; w++) total += stat[w][threadIdx.x][1] * __builtin_amdgcn_exp2f((stat[w][threadIdx.x][0] - to) * to_log2);
		inverse[threadIdx.x] = total == 0.f ? 0.f : 1.f / total;
		if(place.ok) {
			if(a.splits > 1) {
				float* const st = a.part_stat + 2 * ((2 * (int64_t)split + i) * n_rows + first_row + row);
				st[0] = to, st[1] = total;
			} else if(p.stats) {
				float* const st = p.stats + 2 * ((b * 2 * p.H + 2 * place.h + i) * p.Lq + place.qi);
				st[0] = to, st[1] = total == 0.f ? 0.f : 1.f / total;
			}
		}
	}
	// As many columns at a time through LDS as a tile of V has room for; a thread then has two of them of one row, in both maps.
	constexpr int PAIRS = 16 * S::AT_ONCE;
	float* const  mine = reinterpret_cast<float*>(smem) + wave * (S::TABLE / 4) + (lane & 31) * S::LINE + 16 * half;
#pragma unroll
	for(int db = 0; db < TV::BLOCKS; db += S::AT_ONCE) {
		if(32 * db >= Dv) break;
		if(db > 0) __syncthreads();
		if(at_row.ok) {
#pragma unroll
			for(int j = 0; j < S::AT_ONCE; j++)
#pragma unroll
				for(int e = 0; e < 4; e++)
					*reinterpret_cast<f32x4*>(mine + 32 * j + 4 * e) = f32x4{o[db + j][4 * e] * by, o[db + j][4 * e + 1] * by, o[db + j][4 * e + 2] * by, o[db + j][4 * e + 3] * by};
		}
		__syncthreads();
		for(int n = threadIdx.x; n < (int)rows * PAIRS; n += THREADS) {
			const int          row = n / PAIRS, column = 2 * (n - row * PAIRS);
			const float* const all = reinterpret_cast<const float*>(smem) + row * S::LINE + column;
			const row_place    place(row, rows, G, hk);
			const float        lam = a.splits > 1 ? 0.f : lam_of(p, place.h);
#pragma unroll
			for(int c = 0; c < 2; c++) {
				const int at = 32 * db + column + c;
				if(at >= Dv) continue;
				float r[2] = {0.f, 0.f};
#pragma unroll
				for(int i = 0; i < 2; i++)
#pragma unroll
					for(int w = 0; w < WAVES; w++) r[i] += all[w * (S::TABLE / 4) + 16 * i * S::LINE + c];
				if(a.splits > 1) {
#pragma unroll
					for(int i = 0; i < 2; i++) a.part_out[((2 * (int64_t)split + i) * n_rows + first_row + row) * Dv + at] = r[i];
				} else {
					// (no live key: zeros, whatever lam is and whatever V holds at other rows' keys)
					const float second = inverse[16 + row] == 0.f ? 0.f : r[1] * inverse[16 + row], out = inverse[row] == 0.f ? 0.f : __builtin_fmaf(-lam, second, r[0] * inverse[row]);
					store_result<T>(p, b, place.h, place.qi, (b * p.H + place.h) * p.Lq + place.qi, at, out, second);
				}
			}
		}
	}
}

// The parts of the key axis joined: a workgroup per query row; two wavefronts to a map, half of the parts each, four columns to a lane.  The parts' maxima and sums come one to a
// lane (64 parts at most), so that the parts' results, 16 of them in flight, wait for nothing but each other.
constexpr int MAX_PARTS = 64;
template <typename T>
__global__ void __launch_bounds__(THREADS) diff_join_kernel(forward_args a) {
	const af3_diff_attention_params& p = a.p;
	__shared__ f32x4 joint[2][64];
	__shared__ f32x4 halves[2][64];
	const int64_t G = p.H / p.Hkv, rows = G * p.Lq, n_rows = p.B * p.Hkv * rows, at = blockIdx.x;
	const int     lane = threadIdx.x & 63, wave = threadIdx.x >> 6, map = wave & 1, Dv = (int)p.Dv, splits = (int)a.splits;
	const int64_t   bh = at / rows, hk = bh % p.Hkv, b = bh / p.Hkv;
	const row_place place(at - bh * rows, rows, G, hk);
	float m = 0.f, l = 0.f;
	if(lane < splits) m = a.part_stat[2 * ((2 * lane + map) * n_rows + at)], l = a.part_stat[2 * ((2 * lane + map) * n_rows + at) + 1];
	float top = l == 0.f ? LOWEST : m;
#pragma unroll
	for(int d = 32; d; d >>= 1) top = maximum(top, __shfl_xor(top, d));
	const float weight = l == 0.f ? 0.f : __builtin_amdgcn_exp2f((m - top) * a.factor);
	float sum = l * weight;
#pragma unroll
	for(int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
	const float inv = sum == 0.f ? 0.f : 1.f / sum;
	const int   c = 4 * lane, per = (splits + 1) / 2, first = (wave >> 1) * per, end = first + per < splits ? first + per : splits;
	f32x4       o = {0.f, 0.f, 0.f, 0.f};
	const bool    whole = Dv % 4 == 0;   // (lanes behind the last column read what lane 0 does)
	const float* const from = a.part_out + (map * n_rows + at) * Dv + (whole && c >= Dv ? 0 : c);
	for(int s0 = first; s0 < end; s0 += 16) {
		f32x4 x[16];
#pragma unroll
		for(int s = 0; s < 16; s++) {
			const float* const part = from + (s0 + s < end ? s0 + s : end - 1) * (2 * n_rows * Dv);
			if(whole) x[s] = *reinterpret_cast<const f32x4*>(part);
			else
#pragma unroll
				for(int e = 0; e < 4; e++) x[s][e] = c + e < Dv ? part[e] : 0.f;
		}
#pragma unroll
		for(int s = 0; s < 16; s++) {
			const float w = s0 + s < end ? __shfl(weight, (s0 + s) & 63) : 0.f;
#pragma unroll
			for(int e = 0; e < 4; e++) o[e] = w == 0.f ? o[e] : __builtin_fmaf(x[s][e], w, o[e]);   // (a part without a live key wrote nothing)
		}
	}
	if(wave >> 1) halves[map][lane] = o;
	__syncthreads();
	if(wave >> 1) return;
	o += halves[map][lane];
#pragma unroll
	for(int e = 0; e < 4; e++) o[e] *= inv;
	if(p.stats && lane == 0) {
		float* const st = p.stats + 2 * ((b * 2 * p.H + 2 * place.h + map) * p.Lq + place.qi);
		st[0] = top, st[1] = inv;
	}
	joint[map][lane] = o;
	__syncthreads();
	if(map) return;
	const float lam = lam_of(p, place.h);
	const f32x4 second = joint[1][lane];
	for(int e = 0; e < 4; e++)
		if(c + e < Dv) store_result<T>(p, b, place.h, place.qi, (b * p.H + place.h) * p.Lq + place.qi, c + e, sum == 0.f ? 0.f : __builtin_fmaf(-lam, second[e], o[e]), second[e]);
}

// ---- host side -------------------------------------------------------------------------------------------------------------
int width(const af3_diff_attention_params& p) {   // columns of a map's queries and keys that a kernel has, half of those of its values
	const int64_t d = p.D > (p.Dv + 1) / 2 ? p.D : (p.Dv + 1) / 2;
	return d <= 32 ? 32 : d <= 64 ? 64 : 128;
}
// the most wavefronts that can share rows: four where the tiles of 128 keys leave registers and LDS for the rest
template <typename T, int DP>
constexpr int MOST_SHARING = DP * (int)sizeof(T) <= 128 ? 4 : 2;
int most_sharing(const af3_diff_attention_params& p) { return width(p) * (p.dtype == AF3_F32 ? 4 : 2) <= 128 ? 4 : 2; }

int64_t value_tiles(const af3_diff_attention_params& p) { return (p.Lk + value_rows(width(p)) - 1) / value_rows(width(p)); }

struct plan {
	int      kw;
	uint32_t row_tiles, splits;
	int64_t  part;
	bool     half;    // V as fp16
	bool     token;   // diff_token_kernel
};
constexpr int TOKEN_ROWS = 16;
// As parts_for, down to parts of a single step: what a step costs is its way from memory.
int64_t token_parts(const af3_diff_attention_params& p, int64_t groups, int64_t steps, double step_us) {
	constexpr double JOIN_US = 6.0, BYTES_PER_US = 2e6;
	double           best = 0.0;
	int64_t          parts = 1;
	for(int64_t n = 1; n <= MAX_PARTS && n <= steps && (n == 1 || groups * n <= 512); n++) {
		const double us = (double)((steps + n - 1) / n) * step_us + (n > 1 ? JOIN_US + n * 16.0 * p.B * p.H * p.Lq * p.Dv / BYTES_PER_US : 0.0);
		if(n == 1 || us < best) best = us, parts = n;
	}
	return parts;
}
plan forward_plan(const af3_diff_attention_params& p) {
	plan          f;
	const int64_t rows = p.H / p.Hkv * p.Lq, groups = p.B * p.Hkv;
	const bool    fp32 = p.dtype == AF3_F32;
	const int     wide = width(p);
	const int64_t slots = wide * (fp32 ? 4 : 2) <= 64 ? 512 : 256;
	f.token = rows <= TOKEN_ROWS, f.half = false;
	if(f.token) {
		// (128 keys to a step of the workgroup; two workgroups to a compute unit)
		const int64_t steps = (p.Lk + 127) / 128, splits = token_parts(p, groups, steps, (0.9 + 0.018 * wide) * (fp32 ? 2.5 : 1.0));
		const int64_t each = (steps + splits - 1) / splits;
		f.kw = 4, f.row_tiles = 1, f.part = 128 * each, f.splits = (uint32_t)((steps + each - 1) / each);
		return f;
	}
	auto          busy = [&](int kw) { return (rows + 128 / kw - 1) / (128 / kw) * groups; };
	f.kw = rows <= 32 || busy(4) <= slots ? 4 : rows <= 64 || busy(2) <= slots ? 2 : 1;
	if(f.kw > most_sharing(p)) f.kw = most_sharing(p);
	f.row_tiles = (uint32_t)(busy(f.kw) / groups);
	// (V's way through memory and back is worth it where many rows read it: from four tiles of them on.  Without and with it, 128 pairs (four tiles: 128, two and three: 256) of D = 64, over 256,
	// 1024 and 4096 keys: two tiles 39 and 44, 104 and 106, 375 and 373 us; three 52 and 55, 143 and 136, 545 and 500; four 35 and 39, 96 and 90, 359 and 313; eight 66 and 64, 186 and 160, 694
	// and 565.  D = 128, four: 68 and 71, 178 and 171, 659 and 591.)
	f.half = !fp32 && f.kw == 1 && f.row_tiles >= 4 && groups * value_tiles(p) <= 0xffffff;
	const int64_t kt = tile_keys(wide * (fp32 ? 4 : 2), f.kw), key_tiles = (p.Lk + kt - 1) / kt;
	const double  tile_us = (0.4 + 0.033 * wide) * (f.kw == 4 ? 1.0 : 0.6) * (fp32 ? 3.0 : 1.0);
	const int64_t splits = parts_for(busy(f.kw), slots, key_tiles, tile_us, 8.0 * p.B * p.H * p.Lq * p.Dv, MAX_PARTS);
	const int64_t per = (key_tiles + splits - 1) / splits;
	f.part   = per * kt;
	f.splits = (uint32_t)((key_tiles + per - 1) / per);
	return f;
}

template <typename T, int DP, int KW, bool HALF = false>
int launch_forward(const forward_args& a, uint32_t grid, hipStream_t s) {
	using S = forward_shape<T, DP, KW>;
	auto kernel = &diff_forward_kernel<T, DP, KW, HALF>;
	if(S::LDS > 65536 - 8192 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS) != hipSuccess) {
		(void)hipGetLastError();
		return AF3_ERR_LAUNCH;
	}
	hipLaunchKernelGGL(kernel, dim3(grid), dim3(NT), S::LDS, s, a);
	return launch_status();
}
template <typename T, int DP>
int launch_forward_form(const forward_args& a, int kw, uint32_t grid, hipStream_t s) {
	if constexpr(MOST_SHARING<T, DP> == 4)
		if(kw == 4) return launch_forward<T, DP, 4>(a, grid, s);
	if constexpr(sizeof(T) == 2)
		if(a.values) {
			hipLaunchKernelGGL(diff_values_kernel<DP>, dim3((uint32_t)(a.p.B * a.p.Hkv * value_tiles(a.p))), dim3(THREADS), 0, s, a);
			const int rc = launch_status();
			return rc != AF3_OK ? rc : launch_forward<T, DP, 1, true>(a, grid, s);
		}
	return kw == 2 ? launch_forward<T, DP, 2>(a, grid, s) : launch_forward<T, DP, 1>(a, grid, s);
}
template <typename T, int DP>
int launch_token(const forward_args& a, uint32_t grid, hipStream_t s) {
	using S = token_shape<T, DP>;
	auto kernel = &diff_token_kernel<T, DP>;
	if(S::LDS > 65536 - 8192 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS) != hipSuccess) {
		(void)hipGetLastError();
		return AF3_ERR_LAUNCH;
	}
	hipLaunchKernelGGL(kernel, dim3(grid), dim3(THREADS), S::LDS, s, a);
	return launch_status();
}
template <typename T>
int launch_forward_type(const forward_args& a, const plan& f, uint32_t grid, hipStream_t s) {
	const int wide = width(a.p), kw = f.kw;
	if(f.token) {
		if(wide == 32) return launch_token<T, 32>(a, grid, s);
		if constexpr(sizeof(T) == 2)
			if(wide == 128) return launch_token<T, 128>(a, grid, s);
		return launch_token<T, 64>(a, grid, s);
	}
	if(wide == 32) return launch_forward_form<T, 32>(a, kw, grid, s);
	if constexpr(sizeof(T) == 2)
		if(wide == 128) return launch_forward_form<T, 128>(a, kw, grid, s);
	return launch_forward_form<T, 64>(a, kw, grid, s);
}

int64_t values_bytes(const af3_diff_attention_params& p, const plan& f) { return f.half ? p.B * p.Hkv * value_tiles(p) * value_rows(width(p)) * 4 * width(p) : 0; }
int64_t units_bytes(const af3_diff_attention_params& p, const plan& f) { return f.half ? (p.B * p.Hkv * value_tiles(p) + 3) / 4 * 16 : 0; }
packing pack_inputs(af3_diff_attention_params& p, int32_t& columns, int32_t& v_columns, void* space) {
	packing k(p.dtype == AF3_F32 ? 4 : 2);
	columns = k.add(p.q, p.q_stride, p.B, 2 * p.H, p.Lq, p.D, space);
	k.add(p.k, p.k_stride, p.B, 2 * p.Hkv, p.Lk, p.D, space);
	v_columns = k.add(p.v, p.v_stride, p.B, p.Hkv, p.Lk, p.Dv, space);
	return k;
}
int64_t packed_bytes(af3_diff_attention_params p) {
	int32_t columns;
	return pack_inputs(p, columns, columns, nullptr).bytes;
}
int64_t forward_workspace(const af3_diff_attention_params& p, const plan& f) {
	return packed_bytes(p) + (f.splits > 1 ? (int64_t)f.splits * p.B * p.H * p.Lq * (p.Dv + 2) * 8 : 0) + values_bytes(p, f) + units_bytes(p, f);
}

}  // namespace diff

// whether the gradients of k and v can be launched: workgroups of 32 keys, times 256 threads, inside 32 bits
bool diff_gradients_fit(const af3_diff_attention_params& p) { return p.B * p.Hkv * ((p.Lk + 31) / 32) <= 0xffffff; }

int validate_diff_attention(const af3_diff_attention_params* p) {
	if(!p) return AF3_ERR_NULL_POINTER;
	if((p->dtype != AF3_F32 && p->dtype != AF3_BF16) || (p->lam_dtype != AF3_F32 && p->lam_dtype != AF3_BF16)) return AF3_ERR_BAD_DTYPE;
	if(p->B <= 0 || p->H <= 0 || p->Hkv <= 0 || p->Lq <= 0 || p->Lk <= 0 || p->D <= 0 || p->Dv <= 0 || p->H % p->Hkv != 0) return AF3_ERR_BAD_SHAPE;
	if(p->D > (p->dtype == AF3_F32 ? 64 : 128) || p->Dv > (p->dtype == AF3_F32 ? 128 : 256)) return AF3_ERR_UNSUPPORTED_D;
	// (row numbers and the parts' sizes stay far inside 63 bits, a launch's workgroups times their threads inside 32)
	if(p->B > 0xffffff || p->H > 0x7fff || p->Lq > 0x3fffffff || p->Lk > 0x3fffffff || p->B * p->H > 0xffffff || p->B * p->Hkv > 0x7fffff || p->H * p->Lq > 0x3fffffff || p->B * p->H * ((p->Lq + 31) / 32) > 0xffffff) return AF3_ERR_BAD_SHAPE;
	if(p->stats && !diff_gradients_fit(*p)) return AF3_ERR_BAD_SHAPE;   // (they are for a gradient that would be refused)
	if(!p->q || !p->k || !p->v || !p->lam || !p->out || (p->stats != nullptr) != (p->second != nullptr) || (p->residuals && !p->second)) return AF3_ERR_NULL_POINTER;
	if(p->residuals && p->dtype != AF3_BF16) return AF3_ERR_BAD_DTYPE;   // (nothing would be written there)
	for(int i = 0; i < 3; i++)
		if(p->q_stride[i] < 0 || p->k_stride[i] < 0 || p->v_stride[i] < 0 || p->out_stride[i] < 0) return AF3_ERR_BAD_STRIDE;
	// (inputs may repeat rows, results may not)
	if((p->Lq > 1 && p->out_stride[2] < p->Dv) || (p->H > 1 && p->out_stride[1] == 0) || (p->B > 1 && p->out_stride[0] == 0) || p->lam_stride < 0) return AF3_ERR_BAD_STRIDE;
	if(p->key_mask && p->key_mask_stride_b < 0) return AF3_ERR_BAD_STRIDE;
	if(!(p->softmax_scale > 0.f) || !(p->softmax_scale < INFINITY) || p->q_offset >= (int64_t)1 << 40 || p->q_offset <= -((int64_t)1 << 40)) return AF3_ERR_BAD_ARGUMENT;
	return AF3_OK;
}

}  // namespace af3

using namespace af3;

extern "C" int64_t af3_diff_attention_workspace_bytes(const af3_diff_attention_params* params) {
	const int rc = validate_diff_attention(params);
	return rc != AF3_OK ? rc : diff::forward_workspace(*params, diff::forward_plan(*params));
}

extern "C" int af3_diff_attention_forward(const af3_diff_attention_params* params, void* hip_stream) {
	if(const int rc = validate_diff_attention(params); rc != AF3_OK) return rc;
	const diff::plan f = diff::forward_plan(*params);
	if(const int64_t need = diff::forward_workspace(*params, f); need > 0 && (!params->workspace || params->workspace_bytes < need || (reinterpret_cast<uintptr_t>(params->workspace) & 15))) return AF3_ERR_BAD_ARGUMENT;
	if(const int dc = current_device_status(); dc != AF3_OK) return dc;
	const hipStream_t  s = static_cast<hipStream_t>(hip_stream);
	diff::forward_args a;
	const bool         fp32 = params->dtype == AF3_F32;
	a.p = *params, a.row_tiles = f.row_tiles, a.splits = f.splits, a.part = f.part;
	a.factor = params->softmax_scale * LOG2E;
	unsigned char* space = static_cast<unsigned char*>(params->workspace);
	const diff::packing pack = diff::pack_inputs(a.p, a.columns, a.v_columns, space);
	space += pack.bytes;
	const int64_t n_rows = params->B * params->H * params->Lq;
	a.values   = f.half ? space : nullptr, a.units = reinterpret_cast<float*>(space + diff::values_bytes(*params, f));
	a.part_out = reinterpret_cast<float*>(space + diff::values_bytes(*params, f) + diff::units_bytes(*params, f)), a.part_stat = a.part_out + 2 * f.splits * n_rows * params->Dv;
	const uint32_t grid = (uint32_t)(params->B * params->Hkv) * f.row_tiles * f.splits;
	int rc = pack.launch(s);
	if(rc != AF3_OK) return rc;
	rc = fp32 ? diff::launch_forward_type<float>(a, f, grid, s) : diff::launch_forward_type<uint16_t>(a, f, grid, s);
	if(rc != AF3_OK || f.splits == 1) return rc;
	if(fp32) hipLaunchKernelGGL(diff::diff_join_kernel<float>, dim3((uint32_t)n_rows), dim3(cross::THREADS), 0, s, a);
	else hipLaunchKernelGGL(diff::diff_join_kernel<uint16_t>, dim3((uint32_t)n_rows), dim3(cross::THREADS), 0, s, a);
	return launch_status();
}
