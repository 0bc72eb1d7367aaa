// Attention of queries to states of another length: out = softmax(scale q.k^T + bias, mask) . v for q [B, H, Lq, D] and k, v
// [B, Hkv, Lk, D], H a multiple of Hkv (G = H / Hkv query heads share a key head), bf16 or fp32.  af3_cross_attention_forward.
//
// Per 32 query rows and 32 keys:  S^T[key][row] = K . Q^T   (A = K rows from LDS, B = Q in registers),
//                                 O^T[d][row]  += V^T . P^T  (A = V columns from LDS, B = P as the registers of S^T hold it).
// A lane holds one query row (the half-waves 16 keys each), so that the running maximum and sum of the softmax are one register each.
// The G query heads of a key head are one matrix of G * Lq rows: each tile of K and V is read once for all of them.
#include "cross_tiles.hpp"

#include <math.h>

namespace af3 {
namespace cross {

struct forward_args {
	af3_cross_attention_params p;
	uint32_t row_tiles, splits;    // workgroups per (batch, key head); parts of the key axis
	int64_t  part;                 // keys per part, a multiple of SEGMENT or of the tile
	float    factor;               // exp2((t - max) * factor) with t = q.k (no bias) or scale q.k + bias
	int32_t  whole;                // D is a whole number of 16-byte pieces
	float*   part_out;             // [splits][B * Hkv * G * Lq][D] and ...
	float*   part_stat;            // ... [splits][B * Hkv * G * Lq][2] (maximum, sum); maximum -inf: no live key in the part
};

// what a result loses by its rounding to bf16, itself as bf16: the gradient's delta then has the result to 16 bits
template <typename T>
__device__ __forceinline__ void store_residual(const af3_cross_attention_params& p, int64_t row, int d, const float (&v)[16]) {
	if constexpr(sizeof(T) == 2) {
		if(!p.out_residual) return;
		float r[16];
#pragma unroll
		for(int i = 0; i < 16; i++) r[i] = v[i] - kind<T>::value(kind<T>::bits(v[i]));
		store_row16(static_cast<T*>(p.out_residual) + row, d, (int)p.D, r);
	}
}

// KW: wavefronts that share 32 query rows and each take 32 keys of a tile (1: a wavefront takes all 64 keys of one)
template <typename T, int DP, int KW>
struct forward_shape {
	static constexpr int KT = KW == 4 ? 128 : 64, SUB = KT / (32 * KW), ROWS = 32 * (WAVES / KW);
	static constexpr int TILE = KT * tile<T, DP>::STRIDE;
	static constexpr int BUFFERS = 4 * TILE <= 81920 ? 2 : 1;
	static constexpr int JOIN = KW > 1 ? WAVES * 32 * (DP + 4) * 4 : 0;   // the wavefronts' results on their way to each other
	static constexpr int LDS = 2 * BUFFERS * TILE > JOIN ? 2 * BUFFERS * TILE : JOIN;
	// q, the result's sums and the tiles on their way
	static constexpr int REGISTERS = 4 * tile<T, DP>::STEPS + DP / 2 + 8 * passage<T, DP, KT>::N;
};

template <typename T, int DP, int KW, bool BIAS>
__global__ void __launch_bounds__(THREADS, wavefronts(forward_shape<T, DP, KW>::REGISTERS + (BIAS ? 24 : 0))) cross_forward_kernel(forward_args a) {
	using S  = forward_shape<T, DP, KW>;
	using TL = tile<T, DP>;
	constexpr int E = kind<T>::E, KT = S::KT;
	const af3_cross_attention_params& p = a.p;
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ live_keys<KT> live;
	__shared__ float         stat[WAVES][32][2];

	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
	const int kwave = wave % KW, rwave = wave / KW;
	const share    own((uint32_t)blockIdx.x, (uint32_t)(p.B * p.Hkv), a.row_tiles * a.splits);
	const uint32_t split = own.piece / a.row_tiles, row_tile = own.piece - split * a.row_tiles;
	const int64_t  b = own.pair / (uint32_t)p.Hkv, hk = own.pair - (uint32_t)b * (uint32_t)p.Hkv;
	const int64_t G = p.H / p.Hkv, rows = G * p.Lq;
	const int     D = (int)p.D;

	const int64_t R  = (int64_t)row_tile * S::ROWS + 32 * rwave + (lane & 31);
	const bool    ok = R < rows;
	const int64_t g = ok ? R / p.Lq : 0, qi = ok ? R - g * p.Lq : 0, h = hk * G + g;
	u32x4 qf[TL::STEPS];
	load_operand<T, DP>(qf, static_cast<const T*>(p.q) + b * p.q_stride[0] + h * p.q_stride[1] + qi * p.q_stride[2], ok, D, lane);
	const T* const kb = static_cast<const T*>(p.k) + b * p.k_stride[0] + hk * p.k_stride[1];
	const T* const vb = static_cast<const T*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[1];
	const T* const bias = BIAS ? static_cast<const T*>(p.bias) + h * p.bias_stride[0] + qi * p.bias_stride[1] : nullptr;
	const uint8_t* const mask = p.key_mask ? p.key_mask + b * p.key_mask_stride_b : nullptr;

	// p = exp2(t * to_log2 - reference): t = q.k or scale q.k + bias, `reference` = to_log2 * (a maximum of the row's logits so far)
	const float to_log2 = a.factor;
	float  m = LOWEST, reference = -INFINITY, l = 0.f;
	f32x16 o[TL::BLOCKS];
#pragma unroll
	for(int db = 0; db < TL::BLOCKS; db++) o[db] = f32x16{};
	bool any = false, moves = true;   // a live key was met; the reference moves at the next block (the first one, and while a row is far)

	const int64_t last = (int64_t)(split + 1) * a.part < p.Lk ? (int64_t)(split + 1) * a.part : p.Lk;
	const typename TL::reader at(lane);
	passage<T, DP, KT> pk, pv;
	pk.begin(kb, p.k_stride[2], D, a.whole);
	pv.begin(vb, p.v_stride[2], D, a.whole);
	int buffer = 0;
	for(int64_t first = (int64_t)split * a.part; first < last; first += SEGMENT) {
		const int64_t end = first + SEGMENT < last ? first + SEGMENT : last;
		live.scan(mask, first, end);
		int t = live.next(0);
		if(t < 0) continue;
		any = true;
		pk.load(first + (int64_t)t * KT, end);
		pv.load(first + (int64_t)t * KT, end);
		u32x4 bs[S::SUB][16 / E], coming[S::SUB][16 / E];   // biases of this tile and of the one behind it
		auto  fetch_bias = [&](u32x4(&to)[S::SUB][16 / E], int tile_no) {
			if constexpr(BIAS) {
#pragma unroll
				for(int s = 0; s < S::SUB; s++) load_row16_raw(to[s], bias, first + (int64_t)tile_no * KT + 32 * (kwave * S::SUB + s) + 16 * half, p.Lk);
			}
		};
		fetch_bias(coming, t);
		while(t >= 0) {
			if constexpr(BIAS) {
#pragma unroll
				for(int s = 0; s < S::SUB; s++)
#pragma unroll
					for(int i = 0; i < 16 / E; i++) bs[s][i] = coming[s][i];
			}
			unsigned char* const ks = smem + buffer * 2 * S::TILE;
			unsigned char* const vs = ks + S::TILE;
			const tile_bits<KT> bits(live, t);
			const bool          full = bits.full();
			const int following = live.next(t + 1);
			if constexpr(S::BUFFERS == 1) __syncthreads();
			// (what K holds at a dropped key stays in that key's logits, which are not looked at; its row of V meets a weight of zero, and must not be NaN)
			pk.store(ks, true, [](int) { return true; });
			pv.store(vs, full, [&](int row) { return bits.keeps(row); });
			__syncthreads();
			if(following >= 0) {
				pk.load(first + (int64_t)following * KT, end);
				pv.load(first + (int64_t)following * KT, end);
				fetch_bias(coming, following);
			}
#pragma unroll
			for(int s = 0; s < S::SUB; s++) {
				const int      block = kwave * S::SUB + s;
				const uint32_t keep = bits.of_block(block);
				if(keep == 0u) continue;
				float x[16];
				auto  logits = [&] {
					f32x16 acc{};
#pragma unroll
					for(int i = 0; i < TL::STEPS; i++) acc = kind<T>::mma(TL::row_frag(ks, 32 * block, i, at), qf[i], acc);
#pragma unroll
					for(int r = 0; r < 16; r++) x[r] = BIAS ? __builtin_fmaf(acc[r], p.softmax_scale, kind<T>::at(bs[s][r / E], r % E)) : acc[r];
					if(keep != ~0u) drop_keys(x, keep, -INFINITY);
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
				// Optimistic: the probabilities against the reference as it is.  It moves, to the maximum, at a wavefront's first block and where they get large, and
				// then nothing needs a factor until they get large again.
				float sum = 0.f;
				logits();
				if(!moves) {
					sum   = probabilities();
					moves = __any(!(sum < LARGE));
					if(moves) logits();
				}
				if(moves) {
					float top = x[0];
#pragma unroll
					for(int r = 1; r < 16; r++) top = maximum(top, x[r]);
					const float to = maximum(m, maximum_of_halves(top)), by = __builtin_amdgcn_exp2f((m - to) * to_log2);
					m = to, reference = m * to_log2, l *= by;
#pragma unroll
					for(int db = 0; db < TL::BLOCKS; db++) o[db] *= by;
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
#pragma unroll
				for(int j = 0; j < TL::JOINTS; j++) {
					const u32x4 pf = kind<T>::pack(x + E * j);
#pragma unroll
					for(int db = 0; db < TL::BLOCKS; db++) o[db] = kind<T>::mma(TL::col_frag(vs, 32 * block, db, j, at), pf, o[db]);
				}
			}
			t = following;
			if constexpr(S::BUFFERS == 2) buffer ^= 1;
		}
	}
	l = sum_of_halves(l);

	const int64_t bh = b * p.Hkv + hk, n_rows = p.B * p.Hkv * rows;
	if(!any) {
		// No live key here.  Where the batch row has one elsewhere that is all; where it has none, its result is the mean of the values: this part's sum
		// of them, which is the same for all rows.
		if(a.splits > 1) {
			bool elsewhere = false;
			for(int64_t key = threadIdx.x; key < p.Lk; key += THREADS) elsewhere = elsewhere || mask[key] != 0;   // (no mask: there is a live key)
			if(__syncthreads_or(elsewhere)) {
				if(ok && kwave == 0 && half == 0) a.part_stat[2 * (split * n_rows + bh * rows + R)] = -INFINITY, a.part_stat[2 * (split * n_rows + bh * rows + R) + 1] = 0.f;
				return;
			}
		}
		const int64_t first = (int64_t)split * a.part;
		float* const  sums = reinterpret_cast<float*>(smem);   // [THREADS / DP][DP]
		constexpr int PARTS = THREADS / DP;
		const int     d = threadIdx.x % DP, part = threadIdx.x / DP;
		float         sum = 0.f;
		if(part < PARTS && d < D) {
#pragma unroll 4
			for(int64_t key = first + part; key < last; key += PARTS) sum += kind<T>::value(vb[key * p.v_stride[2] + d]);
		}
		if(part < PARTS) sums[part * DP + d] = sum;
		__syncthreads();
		if(!ok || kwave != 0) return;
		const int64_t place = split * n_rows + bh * rows + R;
		if(a.splits > 1 && half == 0) a.part_stat[2 * place] = -INFINITY, a.part_stat[2 * place + 1] = (float)(last - first);
		T* const out = static_cast<T*>(p.out) + b * p.out_stride[0] + h * p.out_stride[1] + qi * p.out_stride[2];
		for(int db = 0; db < TL::BLOCKS; db++) {
			float v[16];
			for(int r = 0; r < 16; r++) {
				v[r] = 0.f;
				for(int i = 0; i < PARTS; i++) v[r] += sums[i * DP + 32 * db + 16 * half + r];
			}
			if(a.splits > 1) {
				store_row16(a.part_out + place * D, 32 * db + 16 * half, D, v);
				continue;
			}
			for(int r = 0; r < 16; r++) v[r] /= (float)p.Lk;
			store_row16(out, 32 * db + 16 * half, D, v);
			store_residual<T>(p, ((b * p.H + h) * p.Lq + qi) * D, 32 * db + 16 * half, v);
		}
		if(p.stats && half == 0 && a.splits == 1) {
			float* const st = p.stats + 2 * ((b * p.H + h) * p.Lq + qi);
			st[0] = -INFINITY, st[1] = 1.f / (float)p.Lk;
		}
		return;
	}

	if constexpr(KW > 1) {   // wavefronts that share rows: each weights its own sums by the common maximum, then a quarter of the columns each
		if(half == 0) stat[wave][lane][0] = m, stat[wave][lane][1] = l;
		__syncthreads();   // (and nobody reads tiles any more)
		float to = LOWEST, sum = 0.f;
#pragma unroll
		for(int w = 0; w < KW; w++) to = maximum(to, stat[rwave * KW + w][lane & 31][0]);
#pragma unroll
		for(int w = 0; w < KW; w++) sum += stat[rwave * KW + w][lane & 31][1] * __builtin_amdgcn_exp2f((stat[rwave * KW + w][lane & 31][0] - to) * a.factor);
		const float by = __builtin_amdgcn_exp2f((m - to) * a.factor);
		m = to, l = sum;
		float* const mine = reinterpret_cast<float*>(smem) + wave * 32 * (DP + 4);
#pragma unroll
		for(int db = 0; db < TL::BLOCKS; db++)
#pragma unroll
			for(int i = 0; i < 4; i++)
				*reinterpret_cast<f32x4*>(mine + (lane & 31) * (DP + 4) + 32 * db + 16 * half + 4 * i) = f32x4{o[db][4 * i] * by, o[db][4 * i + 1] * by, o[db][4 * i + 2] * by, o[db][4 * i + 3] * by};
		__syncthreads();
		const float* const all = reinterpret_cast<const float*>(smem) + rwave * KW * 32 * (DP + 4) + (lane & 31) * (DP + 4) + 16 * half;
#pragma unroll
		for(int db = 0; db < TL::BLOCKS; db++) {
			if(db % KW != kwave) continue;
			o[db] = f32x16{};
#pragma unroll
			for(int w = 0; w < KW; w++)
#pragma unroll
				for(int i = 0; i < 4; i++) {
					const f32x4 v = *reinterpret_cast<const f32x4*>(all + w * 32 * (DP + 4) + 32 * db + 4 * i);
#pragma unroll
					for(int e = 0; e < 4; e++) o[db][4 * i + e] += v[e];
				}
		}
	}
	if(!ok) return;
	const bool first_of_row = kwave == 0 && half == 0;
	if(a.splits > 1) {
		const int64_t place = split * n_rows + bh * rows + R;
		if(first_of_row) a.part_stat[2 * place] = m, a.part_stat[2 * place + 1] = l;
#pragma unroll
		for(int db = 0; db < TL::BLOCKS; db++) {
			if(db % KW != kwave) continue;
			float v[16];
#pragma unroll
			for(int r = 0; r < 16; r++) v[r] = o[db][r];
			store_row16(a.part_out + place * D, 32 * db + 16 * half, D, v);
		}
		return;
	}
	const float inv = l == 0.f ? 0.f : 1.f / l;   // (0: every live key's bias is -inf)
	if(p.stats && first_of_row) {
		float* const st = p.stats + 2 * ((b * p.H + h) * p.Lq + qi);
		st[0] = m, st[1] = inv;
	}
	T* const out = static_cast<T*>(p.out) + b * p.out_stride[0] + h * p.out_stride[1] + qi * p.out_stride[2];
#pragma unroll
	for(int db = 0; db < TL::BLOCKS; db++) {
		if(db % KW != kwave) continue;
		float v[16];
#pragma unroll
		for(int r = 0; r < 16; r++) v[r] = o[db][r] * inv;
		store_row16(out, 32 * db + 16 * half, D, v);
		store_residual<T>(p, ((b * p.H + h) * p.Lq + qi) * D, 32 * db + 16 * half, v);
	}
}

// The parts of the key axis joined: one wavefront per query row, columns over its lanes.  The parts' maxima and sums come one to a lane (64 parts at
// most), so that the parts' results, eight of them in flight, wait for nothing but each other.
constexpr int MAX_PARTS = 64;
template <typename T>
__global__ void __launch_bounds__(THREADS) cross_join_kernel(forward_args a) {
	const af3_cross_attention_params& p = a.p;
	const int64_t G = p.H / p.Hkv, rows = G * p.Lq, n_rows = p.B * p.Hkv * rows;
	const int     lane = threadIdx.x & 63, D = (int)p.D, splits = (int)a.splits;
	const int64_t at = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
	if(at >= n_rows) return;
	const int64_t R = at % rows, bh = at / rows, hk = bh % p.Hkv, b = bh / p.Hkv, g = R / p.Lq, qi = R - g * p.Lq, h = hk * G + g;
	float m = -INFINITY, l = 0.f;
	if(lane < splits) m = a.part_stat[2 * (lane * n_rows + at)], l = a.part_stat[2 * (lane * n_rows + at) + 1];
	float top = m;
#pragma unroll
	for(int i = 32; i; i >>= 1) top = maximum(top, __shfl_xor(top, i));
	// (-inf throughout: no live key in the batch row, and l keys of even weight in a part)
	const bool dead = top == -INFINITY;
	const float weight = dead ? 1.f : m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - top) * a.factor);
	float sum = l * weight;
#pragma unroll
	for(int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
	float o[2] = {0.f, 0.f};
	for(int s0 = 0; s0 < splits; s0 += 8) {
		float x[8][2];
#pragma unroll
		for(int s = 0; s < 8; s++)
#pragma unroll
			for(int k = 0; k < 2; k++) {
				x[s][k] = 0.f;
				if(s0 + s < splits && lane + 64 * k < D) x[s][k] = a.part_out[((s0 + s) * n_rows + at) * D + lane + 64 * k];
			}
#pragma unroll
		for(int s = 0; s < 8; s++) {
			const float w = __shfl(weight, (s0 + s) & 63);
			const bool  none = !dead && __shfl(m, (s0 + s) & 63) == -INFINITY;   // (that part wrote nothing)
#pragma unroll
			for(int k = 0; k < 2; k++) o[k] += none || s0 + s >= splits ? 0.f : x[s][k] * w;
		}
	}
	const float  inv = sum == 0.f ? 0.f : 1.f / sum;
	T* const     out = static_cast<T*>(p.out) + b * p.out_stride[0] + h * p.out_stride[1] + qi * p.out_stride[2];
	const int64_t row = (b * p.H + h) * p.Lq + qi;
#pragma unroll
	for(int k = 0; k < 2; k++)
		if(lane + 64 * k < D) {
			const float v = o[k] * inv;
			out[lane + 64 * k] = kind<T>::bits(v);
			if constexpr(sizeof(T) == 2)
				if(p.out_residual) static_cast<T*>(p.out_residual)[row * D + lane + 64 * k] = kind<T>::bits(v - kind<T>::value(kind<T>::bits(v)));
		}
	if(p.stats && lane == 0) p.stats[2 * row] = dead ? -INFINITY : top, p.stats[2 * row + 1] = inv;
}

// the most wavefronts that can share rows: four, where the tiles of 128 keys leave registers for the rest
template <typename T, int DP>
constexpr int MOST_SHARING = 512 * tile<T, DP>::STRIDE <= 131072 ? 4 : 2;
int most_sharing(const af3_cross_attention_params& p) { return p.dtype == AF3_F32 && p.D > 64 ? MOST_SHARING<float, 128> : 4; }
static_assert(MOST_SHARING<uint16_t, 128> == 4 && MOST_SHARING<float, 64> == 4 && MOST_SHARING<float, 96> == 2 && MOST_SHARING<float, 128> == 2);

// ---- host side -------------------------------------------------------------------------------------------------------------
struct plan {
	int      kw;
	uint32_t row_tiles, splits;
	int64_t  part;
};

// As many wavefronts share rows as leave no more workgroups than fit the chip together, so that a short launch fills it: us of one, two and four sharing, at
// B x H x Lq x Lk x D of 4 x 16 x 384 x 1491 x 64 33.5, 28.2, 40.6 (192, 384 and 768 workgroups), 1 x 16 x 1491 x 4096 x 128 134, 106, 195 (192, 384, 752), 8 x 12 x 512 x 512 x 64
// 18.7, 18.2, 31.9 (384, 768, 1536), 1 x 8 x 1024 x 1024 x 64 19.8, 16.7, 13.6 (64, 128, 256), fp32 4 x 8 x 200 x 768 x 32 38.9, 26.1, 18.0.
plan forward_plan(const af3_cross_attention_params& p) {
	plan          f;
	const int64_t rows = p.H / p.Hkv * p.Lq, groups = p.B * p.Hkv;
	const bool    fp32 = p.dtype == AF3_F32;
	auto          busy = [&](int kw) { return (rows + 128 / kw - 1) / (128 / kw) * groups; };
	f.kw = rows <= 32 || busy(4) <= 512 ? 4 : rows <= 64 || busy(2) <= 512 ? 2 : 1;
	if(f.kw > most_sharing(p)) f.kw = most_sharing(p);
	f.row_tiles = (uint32_t)(busy(f.kw) / groups);
	const int64_t kt = f.kw == 4 ? 128 : 64, key_tiles = (p.Lk + kt - 1) / kt;
	const double  tile_us = (0.4 + 0.011 * p.D) * (f.kw == 4 ? 1.0 : 0.6) * (fp32 ? 3.0 : 1.0);
	const int64_t splits = parts_for(busy(f.kw), p.D > 64 || (fp32 && p.D > 32) ? 256 : 512, key_tiles, tile_us, 4.0 * p.B * p.H * p.Lq * p.D, MAX_PARTS);
	const int64_t per = (key_tiles + splits - 1) / splits;
	f.part   = per * kt;
	f.splits = (uint32_t)((key_tiles + per - 1) / per);
	return f;
}

template <typename T, int DP, int KW, bool BIAS>
int launch_forward(const forward_args& a, uint32_t grid, hipStream_t s) {
	using S = forward_shape<T, DP, KW>;
	auto kernel = &cross_forward_kernel<T, DP, KW, BIAS>;
	if(S::LDS > 65536 - 8192 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS) != hipSuccess) {
		(void)hipGetLastError();
		return AF3_ERR_LAUNCH;
	}
	hipLaunchKernelGGL(kernel, dim3(grid), dim3(THREADS), S::LDS, s, a);
	return launch_status();
}
template <typename T, int DP>
int launch_forward_form(const forward_args& a, int kw, uint32_t grid, hipStream_t s) {
	if constexpr(MOST_SHARING<T, DP> == 4)
		if(kw == 4) return a.p.bias ? launch_forward<T, DP, 4, true>(a, grid, s) : launch_forward<T, DP, 4, false>(a, grid, s);
	if(kw == 2) return a.p.bias ? launch_forward<T, DP, 2, true>(a, grid, s) : launch_forward<T, DP, 2, false>(a, grid, s);
	return a.p.bias ? launch_forward<T, DP, 1, true>(a, grid, s) : launch_forward<T, DP, 1, false>(a, grid, s);
}
template <typename T>
int launch_forward_type(const forward_args& a, int kw, uint32_t grid, hipStream_t s) {
	if(a.p.D <= 32) return launch_forward_form<T, 32>(a, kw, grid, s);
	if(a.p.D <= 64) return launch_forward_form<T, 64>(a, kw, grid, s);
	if(a.p.D <= 96) return launch_forward_form<T, 96>(a, kw, grid, s);
	return launch_forward_form<T, 128>(a, kw, grid, s);
}

int64_t forward_workspace(const af3_cross_attention_params& p, const plan& f) { return f.splits > 1 ? (int64_t)f.splits * p.B * p.H * p.Lq * (p.D + 2) * 4 : 0; }

}  // namespace cross

// whether the gradients of k and v can be launched: workgroups of 32 keys, times 256 threads, inside 32 bits
bool cross_gradients_fit(const af3_cross_attention_params& p) { return p.B * p.Hkv * ((p.Lk + 31) / 32) <= 0xffffff; }

int validate_cross_attention(const af3_cross_attention_params* p) {
	if(!p) return AF3_ERR_NULL_POINTER;
	if(p->dtype != AF3_F32 && p->dtype != AF3_BF16) return AF3_ERR_BAD_DTYPE;
	if(p->B <= 0 || p->H <= 0 || p->Hkv <= 0 || p->Lq <= 0 || p->Lk <= 0 || p->D <= 0 || p->H % p->Hkv != 0) return AF3_ERR_BAD_SHAPE;
	if(p->D > AF3_DPA_MAX_HEAD_DIM) return AF3_ERR_UNSUPPORTED_D;
	// (row numbers and the parts' sizes stay far inside 63 bits, a launch's workgroups times 256 threads inside 32)
	if(p->B > 0xffffff || p->H > 0xffff || p->Lq > 0x3fffffff || p->Lk > 0x3fffffff || p->B * p->H > 0xffffff || p->H * p->Lq > 0x7fffffff || p->B * p->H * ((p->Lq + 31) / 32) > 0xffffff) return AF3_ERR_BAD_SHAPE;
	if(p->stats && !cross_gradients_fit(*p)) return AF3_ERR_BAD_SHAPE;   // (they are for a gradient that would be refused)
	if(!p->q || !p->k || !p->v || !p->out) return AF3_ERR_NULL_POINTER;
	for(int i = 0; i < 3; i++)
		if(p->q_stride[i] < 0 || p->k_stride[i] < 0 || p->v_stride[i] < 0 || p->out_stride[i] < 0) return AF3_ERR_BAD_STRIDE;
	// (inputs may repeat rows, results may not)
	if((p->Lq > 1 && p->out_stride[2] < p->D) || (p->H > 1 && p->out_stride[1] == 0) || (p->B > 1 && p->out_stride[0] == 0)) return AF3_ERR_BAD_STRIDE;
	if(p->bias && (p->bias_stride[0] < 0 || p->bias_stride[1] < 0)) return AF3_ERR_BAD_STRIDE;
	if(p->key_mask && p->key_mask_stride_b < 0) return AF3_ERR_BAD_STRIDE;
	if(!(p->softmax_scale > 0.f) || !(p->softmax_scale < INFINITY)) return AF3_ERR_BAD_ARGUMENT;
	return AF3_OK;
}

}  // namespace af3

using namespace af3;

extern "C" int64_t af3_cross_attention_workspace_bytes(const af3_cross_attention_params* params) {
	const int rc = validate_cross_attention(params);
	return rc != AF3_OK ? rc : cross::forward_workspace(*params, cross::forward_plan(*params));
}

extern "C" int af3_cross_attention_forward(const af3_cross_attention_params* params, void* hip_stream) {
	if(const int rc = validate_cross_attention(params); rc != AF3_OK) return rc;
	const cross::plan f = cross::forward_plan(*params);
	if(const int64_t need = cross::forward_workspace(*params, f); need > 0 && (!params->workspace || params->workspace_bytes < need || (reinterpret_cast<uintptr_t>(params->workspace) & 15))) return AF3_ERR_BAD_ARGUMENT;
	if(const int dc = current_device_status(); dc != AF3_OK) return dc;
	const hipStream_t   s = static_cast<hipStream_t>(hip_stream);
	cross::forward_args a;
	a.p = *params, a.row_tiles = f.row_tiles, a.splits = f.splits, a.part = f.part;
	a.factor = params->bias ? LOG2E : params->softmax_scale * LOG2E;
	a.whole  = params->D * (params->dtype == AF3_F32 ? 4 : 2) % 16 == 0;
	const int64_t n_rows = params->B * params->H * params->Lq;
	a.part_out = static_cast<float*>(params->workspace), a.part_stat = a.part_out + f.splits * n_rows * params->D;
	const uint32_t grid = (uint32_t)(params->B * params->Hkv) * f.row_tiles * f.splits;
	int rc = params->dtype == AF3_F32 ? cross::launch_forward_type<float>(a, f.kw, grid, s) : cross::launch_forward_type<uint16_t>(a, f.kw, grid, s);
	if(rc != AF3_OK || f.splits == 1) return rc;
	const uint32_t joins = (uint32_t)((n_rows + cross::WAVES - 1) / cross::WAVES);
	if(params->dtype == AF3_F32) hipLaunchKernelGGL(cross::cross_join_kernel<float>, dim3(joins), dim3(cross::THREADS), 0, s, a);
	else hipLaunchKernelGGL(cross::cross_join_kernel<uint16_t>, dim3(joins), dim3(cross::THREADS), 0, s, a);
	return launch_status();
}
