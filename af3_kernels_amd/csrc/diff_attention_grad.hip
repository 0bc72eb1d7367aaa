// The gradients of diff_attention.hip's attention.  With P1, P2 the two maps of a head, O2 = P2 . v, dO = the gradient of out = (P1 - lam P2) . v:
//     dv = (P1 - lam P2)^T . dO,  dP = dO . v^T (one product for both maps),  d2 = rowsum(dO * O2),  d1 = rowsum(dO * O1) = rowsum(dO * out) + lam d2,
//     dS1 = P1 * (dP - d1),  dS2 = -lam P2 * (dP - d2),  dq_i = scale dS_i . k_i,  dk_i = scale dS_i^T . q_i,  dlam = -sum of d2 over the head's rows.
// P1 and P2 are computed again from q, k and the two numbers per row and map that the forward pass left.  Kernels, none with atomics: each element of a result is
// summed by one workgroup, or by one per part of the long axis and a joining kernel, always in the same order.
//   diff_delta_kernel d1 and d2
//   diff_dq_kernel    32 query rows per wavefront, both maps, keys in tiles
//   diff_dkv_kernel   32 keys per wavefront, query rows in tiles, over all heads of the key head
//   diff_lam_kernel   the sums of d2, and of the rows of P2 * (dP - d2): those would be zero, but for what d2 misses by the forward pass's probabilities, rounded to bf16 as they are
//                     there.  dlam is a sum of many rows' d2 that mostly cancel: without that it was off by up to 0.008 of itself in sums over 300 rows (with: 1e-6 before its last rounding).
#include "diff_tiles.hpp"
#include "launch_grid.hpp"

#include <math.h>

namespace af3 {
namespace diff {

struct grad_args {
	af3_diff_attention_params p;
	af3_diff_attention_grads  g;
	uint32_t tiles, splits;   // workgroups per (batch, key head), parts of the long axis
	int64_t  part;            // dq: keys per part; dK and dV: tiles of query rows per part
	float    factor;
	int32_t  columns, v_columns;   // of q and k, of v and grad_out, as they are read: whole pieces
	float *  d1, *d2;         // [B, H, Lq] each
	float*   short_of;        // what d2 is short of, in `shorts` parts [B, H, Lq], or null
	uint32_t shorts;
	float*   partial;         // dq: [splits][B 2H Lq][D]; dK and dV: [splits]([B 2Hkv Lk][D], [B Hkv Lk][Dv])
	float *  dq_space, *dkv_space;
};

// the sum of the wavefronts' results of equal shape, wavefront w keeps the blocks of columns that are w modulo N; `tables`: N of 32 x (W + 4)
template <int W, int N>
__device__ __forceinline__ void add_up(float* tables, int w, int lane, f32x16 (&o)[W / 32]) {
	const int at = (lane & 31) * (W + 4) + 16 * (lane >> 5);
	__syncthreads();
#pragma unroll
	for(int db = 0; db < W / 32; db++)
#pragma unroll
		for(int i = 0; i < 4; i++) *reinterpret_cast<f32x4*>(tables + w * 32 * (W + 4) + at + 32 * db + 4 * i) = f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
	__syncthreads();
#pragma unroll
	for(int db = 0; db < W / 32; db++) {
		if(db % N != w) continue;
		o[db] = f32x16{};
#pragma unroll
		for(int k = 0; k < N; k++)
#pragma unroll
			for(int i = 0; i < 4; i++) {
				const f32x4 v = *reinterpret_cast<const f32x4*>(tables + k * 32 * (W + 4) + at + 32 * db + 4 * i);
#pragma unroll
				for(int e = 0; e < 4; e++) o[db][4 * i + e] += v[e];
			}
	}
}

// d1 and d2: 8, 16 or 32 lanes per row, 8 columns each (those of out and of second are read to 16 bits where the forward pass left what their rounding lost)
__host__ __device__ constexpr int delta_lanes(const af3_diff_attention_params& p) { return p.Dv <= 64 ? 8 : p.Dv <= 128 ? 16 : 32; }
template <typename T>
__global__ void __launch_bounds__(THREADS) diff_delta_kernel(grad_args a) {
	const af3_diff_attention_params& p = a.p;
	const int     lanes = delta_lanes(p);
	const int64_t n_rows = p.B * p.H * p.Lq, row = (blockIdx.y * (int64_t)gridDim.x + blockIdx.x) * (THREADS / lanes) + threadIdx.x / lanes;
	if(row >= n_rows) return;   // (all lanes of the row)
	const int64_t bh = (uint32_t)row / (uint32_t)p.Lq, qi = row - bh * p.Lq, b = (uint32_t)bh / (uint32_t)p.H, h = bh - b * p.H;   // (fewer than 2^29 rows)
	const int     lane = threadIdx.x & (lanes - 1), Dv = (int)p.Dv;
	auto eight = [&](const T* from, float (&x)[8]) {
		if(8 * lane + 8 <= Dv) {
			if constexpr(sizeof(T) == 2) {
				const u32x4 v = load16(from + 8 * lane);
#pragma unroll
				for(int e = 0; e < 8; e++) x[e] = kind<T>::at(v, e);
			} else {
				const u32x4 v = load16(from + 8 * lane), w = load16(from + 8 * lane + 4);
#pragma unroll
				for(int e = 0; e < 4; e++) x[e] = kind<T>::at(v, e), x[4 + e] = kind<T>::at(w, e);
			}
		} else {
#pragma unroll
			for(int e = 0; e < 8; e++) {
				x[e] = 0.f;
				if(8 * lane + e < Dv) x[e] = kind<T>::value(from[8 * lane + e]);
			}
		}
	};
	float g[8], o[8], s[8];
	eight(static_cast<const T*>(a.g.grad_out) + b * a.g.grad_out_stride[0] + h * a.g.grad_out_stride[1] + qi * a.g.grad_out_stride[2], g);
	eight(static_cast<const T*>(p.out) + b * p.out_stride[0] + h * p.out_stride[1] + qi * p.out_stride[2], o);
	eight(static_cast<const T*>(p.second) + row * Dv, s);
	if(sizeof(T) == 2 && p.residuals) {
		float x[8], y[8];
		eight(static_cast<const T*>(p.residuals) + row * Dv, x);
		eight(static_cast<const T*>(p.residuals) + (n_rows + row) * Dv, y);
#pragma unroll
		for(int e = 0; e < 8; e++) o[e] += x[e], s[e] += y[e];
	}
	float d1 = 0.f, d2 = 0.f;
#pragma unroll
	for(int e = 0; e < 8; e++) d1 = __builtin_fmaf(g[e], o[e], d1), d2 = __builtin_fmaf(g[e], s[e], d2);
#pragma unroll
	for(int i = 16; i; i >>= 1)
		if(i < lanes) d1 += __shfl_xor(d1, i), d2 += __shfl_xor(d2, i);
	if(lane == 0) a.d1[row] = __builtin_fmaf(lam_of(p, h), d2, d1), a.d2[row] = d2;
}

// How many rows a tile has, how many maps a wavefront and how many threads the kernels, by the bytes of a row of q or k (of 32, 64 or 128 columns).
constexpr int tile_rows(int bytes, int sharing) { return sharing == 4 || bytes <= 64 ? 128 : bytes <= 128 ? 64 : 32; }
constexpr int dq_maps(int bytes) { return bytes <= 128 ? 2 : 1; }
constexpr int DQ_THREADS = 512;
// dK and dV of 128-byte rows: both maps in a wavefront need 370 registers, one wavefront to a SIMD; with one map each, and dP computed by both, there are two (2 x 16 (4) x 4096 x 64
// causal 761 -> 579 us, in workgroups of 256 threads 776; 540 with the tiles dealt out longest first).  Where wavefronts share their keys the pairs' exchange would be between twice as many.
constexpr int dkv_maps(int bytes, int sharing) { return bytes <= 64 || sharing > 1 ? 2 : 1; }
constexpr int dkv_threads(int bytes, int sharing) { return bytes == 128 && sharing == 1 ? 512 : 256; }

// ---- dQ ----
// KW: wavefronts that share 32 rows and each take 32 keys of a tile; MAPS: maps of a wavefront, 2, or 1 with the other map beside it in another one
template <typename T, int DP, int KW>
struct dq_shape {
	static constexpr int BYTES = DP * (int)sizeof(T), MAPS = dq_maps(BYTES), NT = DQ_THREADS, W = NT / 64, GROUPS = W * MAPS / 2 / KW;
	static constexpr int DV = 2 * DP, KT = tile_rows(BYTES, KW), SUB = KT / (32 * KW), ROWS = 32 * GROUPS;
	static constexpr int KTILE = KT * tile<T, DP>::STRIDE, VTILE = KT * tile<T, DV>::STRIDE, SET = 2 * KTILE + VTILE;
	static constexpr int BUFFERS = 2 * SET <= 65536 ? 2 : 1;
	static constexpr int JOIN = KW > 1 ? W * 32 * (DP + 4) * 4 : 0;
	static constexpr int LDS = BUFFERS * SET > JOIN ? BUFFERS * SET : JOIN;
};

template <typename T, int DP, int KW>
__global__ void __launch_bounds__((dq_shape<T, DP, KW>::NT), 2) diff_dq_kernel(grad_args a) {
	using S  = dq_shape<T, DP, KW>;
	using TK = tile<T, DP>;
	using TV = tile<T, S::DV>;
	constexpr int E = kind<T>::E, KT = S::KT, MAPS = S::MAPS;
	const af3_diff_attention_params& p = a.p;
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ live_keys<KT> live;

	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
	const int map0 = MAPS == 2 ? 0 : wave & 1, place = MAPS == 2 ? wave : wave >> 1, kwave = place % KW, group = place / KW;   // (map0: the wavefront's first map)
	const dealt    own((uint32_t)blockIdx.x, (uint32_t)(p.B * p.Hkv), a.tiles, a.splits, p.causal != 0);
	const uint32_t split = own.split, row_tile = a.tiles - 1 - own.tile;
	const int64_t  b = own.pair / (uint32_t)p.Hkv, hk = own.pair - (uint32_t)b * (uint32_t)p.Hkv;
	const int64_t G = p.H / p.Hkv, rows = G * p.Lq;
	const int     D = (int)p.D;

	const int64_t   R = (int64_t)row_tile * S::ROWS + 32 * group + (lane & 31);
	const row_place at_row(R, rows, G, hk);
	const bool      ok = at_row.ok;
	const int64_t   qi = at_row.qi, h = at_row.h, row = (b * p.H + h) * p.Lq + qi;
	u32x4 qf[MAPS][TK::STEPS], gf[TV::STEPS];
#pragma unroll
	for(int i = 0; i < MAPS; i++) load_rows<T, DP>(qf[i], static_cast<const T*>(p.q) + b * p.q_stride[0] + (2 * h + map0 + i) * p.q_stride[1] + qi * p.q_stride[2], ok, a.columns, lane);
	load_rows<T, S::DV>(gf, static_cast<const T*>(a.g.grad_out) + b * a.g.grad_out_stride[0] + h * a.g.grad_out_stride[1] + qi * a.g.grad_out_stride[2], ok, a.v_columns, lane);
	const float d1 = ok ? a.d1[row] : 0.f, d2 = ok ? a.d2[row] : 0.f;
	float delta[MAPS];
	float m[MAPS], inv[MAPS], taken[MAPS];
	bool  far = false;
#pragma unroll
	for(int i = 0; i < MAPS; i++) {
		delta[i] = map0 + i == 0 ? d1 : d2;
		const int64_t at = (b * 2 * p.H + 2 * h + map0 + i) * p.Lq + qi;
		m[i] = ok ? p.stats[2 * at] : 0.f, inv[i] = ok ? p.stats[2 * at + 1] : 0.f;
		taken[i] = whole_reference(m[i], inv[i], a.factor);
		far = far || is_far(m[i] * a.factor);
	}
	const bool apart = sizeof(T) == 4 || __any(far);   // (a row far from zero: in the logits' own units)
	const T* const kb = static_cast<const T*>(p.k) + b * p.k_stride[0] + 2 * hk * p.k_stride[1];
	const T* const vb = static_cast<const T*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[1];
	const uint8_t* const mask = p.key_mask ? p.key_mask + b * p.key_mask_stride_b : nullptr;

	float  row_sum = 0.f;   // of the second map's dS / -lam
	f32x16 dq[MAPS][TK::BLOCKS];
#pragma unroll
	for(int i = 0; i < MAPS; i++)
#pragma unroll
		for(int db = 0; db < TK::BLOCKS; db++) dq[i][db] = f32x16{};

	int64_t last = (int64_t)(split + 1) * a.part < p.Lk ? (int64_t)(split + 1) * a.part : p.Lk;
	if(p.causal) {
		const int64_t end_row = (int64_t)(row_tile + 1) * S::ROWS < rows ? (int64_t)(row_tile + 1) * S::ROWS : rows, end = (end_row - 1) / G + p.q_offset + 1;
		last = end < last ? end : last;
	}
	const int64_t limit = p.causal ? qi + p.q_offset : (int64_t)1 << 41;
	const typename TK::reader at_k_(lane);
	const typename TV::reader at_v_(lane);
	carrier<T, DP, KT, S::NT>    pk[2];
	carrier<T, S::DV, KT, S::NT> pv;
	pk[0].begin(p.k_stride[2], a.columns);
	pv.begin(p.v_stride[2], a.v_columns);
	int buffer = 0;
	for(int64_t first = (int64_t)split * a.part; first < last; first += SEGMENT) {
		const int64_t end = first + SEGMENT < last ? first + SEGMENT : last;
		live.template scan<S::NT>(mask, first, end);
		int t = live.next(0);
		if(t < 0) continue;
		const int within = limit - first > SEGMENT ? SEGMENT : limit - first < -1 ? -1 : (int)(limit - first);
		auto fetch = [&](int tile_no) {
			const int64_t from = first + (int64_t)tile_no * KT;
			pk[0].load(kb, from, end), pk[1].load(kb + p.k_stride[1], from, end, pk[0]), pv.load(vb, from, end);
		};
		fetch(t);
		while(t >= 0) {
			unsigned char* const ks = smem + buffer * S::SET;
			unsigned char* const vs = ks + 2 * S::KTILE;
			const tile_bits<KT> bits(live, t);
			const bool          full = bits.full();
			const int following = live.next(t + 1);
			if constexpr(S::BUFFERS == 1) __syncthreads();
			// (V is only multiplied row by row, and dS of a dropped key is not looked at; K's rows are added up under weights of zero)
			pk[0].store(ks, full, [&](int r) { return bits.keeps(r); });
			pk[1].store(ks + S::KTILE, full, [&](int r) { return bits.keeps(r); }, a.columns);
			pv.store(vs, true, [](int) { return true; });
			__syncthreads();
			if(following >= 0) fetch(following);
#pragma unroll 1
			for(int s = 0; s < S::SUB; s++) {
				const int      block = kwave * S::SUB + s;
				const uint32_t keep  = bits.of_block(block);
				const int      left = within - (t * KT + 32 * block + 16 * half);
				if(keep == 0u || !__any(ok && left >= 0)) continue;
				const typename TK::reader at_k = fresh(at_k_);
				const typename TV::reader at_v = fresh(at_v_);
				const bool diagonal = __any(ok && left < 15);
				f32x16 dp{};
#pragma unroll
				for(int st = 0; st < TV::STEPS; st++) dp = kind<T>::mma(TV::row_frag(vs, 32 * block, st, at_v), gf[st], dp);
#pragma unroll
				for(int i = 0; i < MAPS; i++) {
					const unsigned char* const km = ks + (map0 + i) * S::KTILE;
					f32x16 acc{};
#pragma unroll
					for(int st = 0; st < TK::STEPS; st++) acc = kind<T>::mma(TK::row_frag(km, 32 * block, st, at_k), qf[i][st], acc);
					float x[16];
					if(apart) {
#pragma unroll
						for(int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_exp2f((acc[r] - m[i]) * a.factor) * inv[i] * (dp[r] - delta[i]);
					} else {
#pragma unroll
						for(int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[r], a.factor, -taken[i])) * (dp[r] - delta[i]);
					}
					if(keep != ~0u) drop_keys(x, keep, 0.f);
					if(diagonal) drop_later(x, left, 0.f);
					if(map0 + i == 1) {
#pragma unroll
						for(int r = 0; r < 16; r++) row_sum += x[r];
					}
#pragma unroll
					for(int j = 0; j < TK::JOINTS; j++) {
						const u32x4 f = kind<T>::pack(x + E * j);
#pragma unroll
						for(int db = 0; db < TK::BLOCKS; db++) dq[i][db] = kind<T>::mma(TK::col_frag(km, 32 * block, db, j, at_k), f, dq[i][db]);
					}
				}
			}
			t = following;
			if constexpr(S::BUFFERS == 2) buffer ^= 1;
		}
	}
	row_sum = sum_of_halves(row_sum);
	if(a.short_of && ok && half == 0 && (MAPS == 2 || map0 == 1)) {
		a.short_of[(int64_t)(split * KW + kwave) * (p.B * p.H * p.Lq) + row] = row_sum;
		if(inv[MAPS - 1] == 0.f) a.d2[row] = 0.f;   // (no live key: no part in lam's gradient, whatever its own is; nobody else looks at it)
	}
	if(!a.g.grad_q) return;
	const float lam = lam_of(p, h);
#pragma unroll
	for(int i = 0; i < MAPS; i++) {
		if constexpr(KW > 1) add_up<DP, KW>(reinterpret_cast<float*>(smem) + (MAPS == 2 ? group : 2 * group + map0) * KW * 32 * (DP + 4), kwave, lane, dq[i]);
		if(!ok) continue;
		const float   scale = map0 + i == 0 ? p.softmax_scale : inv[i] == 0.f ? 0.f : -lam * p.softmax_scale;   // (the second map's dS is -lam times what was summed; no live key: zeros, whatever lam is)
		const int64_t to = (b * 2 * p.H + 2 * h + map0 + i) * p.Lq + qi;
#pragma unroll
		for(int db = 0; db < TK::BLOCKS; db++) {
			if(db % KW != kwave) continue;
			float v[16];
#pragma unroll
			for(int r = 0; r < 16; r++) v[r] = dq[i][db][r] * scale;
			if(a.splits > 1) store_columns(a.partial + (split * (p.B * 2 * p.H * p.Lq) + to) * D, 32 * db + 16 * half, D, v);
			else store_columns(static_cast<T*>(a.g.grad_q) + to * D, 32 * db + 16 * half, D, v);
		}
	}
}

// What the kernel with query rows in tiles keeps of each row of a tile in LDS: d1 and d2, and per map the whole reference (bf16), maximum and 1 / sum (fp32 and tiles with
// a row far from zero).  Behind them a word per 64 rows that says whether there is one.  (As a further step of the products instead, three bf16 terms to a number, they were
// no faster, both maps to a wavefront: 236 us for 226 at 4 x 8 (2) x 1491 x 64, 230 for 190 at 4 x 8 x 1024 x 128.)
enum { LESS = 0, TAKEN = 2, MOST = 4, INVERSE = 6, ROW_STATS = 8 };
template <typename T, int QT>
struct row_stats {
	static constexpr int BYTES = ROW_STATS * QT * 4 + 16;
	float v[ROW_STATS];   // of one row, on its way
	// bh: b * H + h; rows are counted from `shift` on, `rows` of them
	__device__ __forceinline__ void load(const grad_args& a, int64_t bh, int q0, int shift, int rows) {
#pragma unroll
		for(int i = 0; i < ROW_STATS; i++) v[i] = 0.f;
		const int qi = q0 + (int)threadIdx.x;
		if((int)threadIdx.x >= QT || qi >= rows) return;
		const int64_t first = bh * a.p.Lq + shift;
		v[LESS] = a.d1[first + qi], v[LESS + 1] = a.d2[first + qi];
#pragma unroll
		for(int i = 0; i < 2; i++) {
			const float* const st = a.p.stats + 2 * (first + bh * a.p.Lq) + 2 * i * a.p.Lq + 2 * qi;
			v[MOST + i] = st[0], v[INVERSE + i] = st[1];
		}
	}
	__device__ __forceinline__ void store(float* st, float factor) {
		if((int)threadIdx.x >= QT) return;
		bool far = false;
#pragma unroll
		for(int i = 0; i < 2; i++) v[TAKEN + i] = whole_reference(v[MOST + i], v[INVERSE + i], factor), far = far || is_far(v[MOST + i] * factor);
#pragma unroll
		for(int i = 0; i < ROW_STATS; i++) st[i * QT + threadIdx.x] = v[i];
		const bool any = __any(far);
		if((threadIdx.x & 63) == 0) reinterpret_cast<int*>(st + ROW_STATS * QT)[threadIdx.x >> 6] = any;
	}
	// whether the rows' maxima and sums are to be taken apart
	static __device__ __forceinline__ bool apart(const float* st) {
		if constexpr(sizeof(T) == 4) return true;
		const int* const far = reinterpret_cast<const int*>(st + ROW_STATS * QT);
		return __builtin_amdgcn_readfirstlane(QT > 64 ? far[0] | far[1] : far[0]) != 0;
	}
	static __device__ __forceinline__ f32x16 sixteen(const float* at) {
		f32x16 x;
#pragma unroll
		for(int i = 0; i < 4; i++) {
			const f32x4 y = *reinterpret_cast<const f32x4*>(at + 4 * i);
			x[4 * i] = y[0], x[4 * i + 1] = y[1], x[4 * i + 2] = y[2], x[4 * i + 3] = y[3];
		}
		return x;
	}
};

// ---- dK, dV ----
// RW: wavefronts that share 32 keys and each take 32 rows of a tile of query rows (1: every wavefront has its own keys and takes the whole tile).  MAPS as in dq_shape.
template <typename T, int DP, int RW>
struct dkv_shape {
	static constexpr int BYTES = DP * (int)sizeof(T), MAPS = dkv_maps(BYTES, RW), NT = dkv_threads(BYTES, RW), W = NT / 64, GROUPS = W * MAPS / 2 / RW;
	static constexpr int DV = 2 * DP, QT = tile_rows(BYTES, RW), SUB = QT / (32 * RW), KEYS = 32 * GROUPS;
	static constexpr int QTILE = QT * tile<T, DP>::STRIDE, GTILE = QT * tile<T, DV>::STRIDE, STATS = row_stats<T, QT>::BYTES, SET = 2 * QTILE + GTILE + STATS;
	static constexpr int BUFFERS = 2 * SET <= 73728 ? 2 : 1;
	// One map to a wavefront: the two of a pair exchange their probabilities, so that their difference is rounded once, and have half of dV's columns each.
	static constexpr int VBLOCKS = DV / 32 * MAPS / 2, EXCHANGE = MAPS == 1 ? SUB * W * 64 * 64 : 0;
	static_assert(MAPS == 2 || RW == 1);
	static constexpr int JOIN = RW > 1 ? W * 32 * (DV + 4) * 4 : 0, PER_SIMD = BYTES <= 64 || (BYTES == 128 && MAPS == 1) ? 2 : 1;   // wavefronts to a SIMD, by the registers of sums and operands
	static constexpr int LDS = BUFFERS * SET + EXCHANGE > JOIN ? BUFFERS * SET + EXCHANGE : JOIN;
};

template <typename T, int DP, int RW>
__global__ void __launch_bounds__((dkv_shape<T, DP, RW>::NT), (dkv_shape<T, DP, RW>::PER_SIMD)) diff_dkv_kernel(grad_args a) {
	using S  = dkv_shape<T, DP, RW>;
	using TK = tile<T, DP>;
	using TV = tile<T, S::DV>;
	constexpr int E = kind<T>::E, QT = S::QT, MAPS = S::MAPS;
	const af3_diff_attention_params& p = a.p;
	constexpr int NONE = 1 << 30;
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ int first_live[S::W];   // of the wavefronts

	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
	const int map0 = MAPS == 2 ? 0 : wave & 1, in_group = MAPS == 2 ? wave : wave >> 1, rwave = in_group % RW, group = in_group / RW;   // (map0: the wavefront's first map)
	const dealt    own((uint32_t)blockIdx.x, (uint32_t)(p.B * p.Hkv), a.tiles, a.splits, p.causal != 0);
	const uint32_t split = own.split, key_tile = own.tile;   // (causal: the first keys have the most rows)
	const int64_t  b = own.pair / (uint32_t)p.Hkv, hk = own.pair - (uint32_t)b * (uint32_t)p.Hkv;
	const int64_t G = p.H / p.Hkv;

	const int64_t key0 = (int64_t)key_tile * S::KEYS, key = key0 + 32 * group + (lane & 31);
	const bool    in = key < p.Lk;
	const bool    lives = in && (!p.key_mask || p.key_mask[b * p.key_mask_stride_b + key] != 0);
	u32x4 kf[MAPS][TK::STEPS], vf[TV::STEPS];
#pragma unroll
	for(int i = 0; i < MAPS; i++) load_rows<T, DP>(kf[i], static_cast<const T*>(p.k) + b * p.k_stride[0] + (2 * hk + map0 + i) * p.k_stride[1] + (in ? key : 0) * p.k_stride[2], in, a.columns, lane);
	load_rows<T, S::DV>(vf, static_cast<const T*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[1] + (in ? key : 0) * p.v_stride[2], in, a.v_columns, lane);
	const uint64_t living = __ballot(lives);
	const bool     work = living != 0;   // (of this wavefront)

	f32x16 dk[MAPS][TK::BLOCKS], dv[S::VBLOCKS];
	const int vblock0 = MAPS == 2 ? 0 : map0 * S::VBLOCKS;   // the wavefront's first block of dV's columns
#pragma unroll
	for(int i = 0; i < MAPS; i++)
#pragma unroll
		for(int db = 0; db < TK::BLOCKS; db++) dk[i][db] = f32x16{};
#pragma unroll
	for(int db = 0; db < S::VBLOCKS; db++) dv[db] = f32x16{};

	// Tiles of query rows, head after head: tile `at` of head `head` of the group, counted head * q_tiles + at (below 2^25).
	const int q_tiles = (int)((p.Lq + QT - 1) / QT), n = (int)G * q_tiles;
	if(lane == 0) first_live[wave] = work ? 32 * group + __builtin_ctzll(living) : NONE;
	__syncthreads();
	int first = first_live[lane % S::W];   // the workgroup's first key that counts, from key0 on
#pragma unroll
	for(int d = S::W / 2; d; d >>= 1) first = min(first, __shfl_xor(first, d));
	first = __builtin_amdgcn_readfirstlane(first);
	// Causal: queries in front of the workgroup's first key that counts have nothing of its keys, and the tiles begin behind them: queries without a key are among them, which have no part
	// in a gradient, and whatever stands there would meet weights of zero, which NaN does not heed.
	const int64_t skipped = p.causal ? key0 + first - p.q_offset : 0;
	const int     skip = skipped <= 0 ? 0 : skipped < p.Lq ? (int)skipped : (int)p.Lq, from = skip / QT, shift = skip - from * QT;
	// (rows are counted from `shift` on in what follows, so that tiles begin at whole numbers of them)
	const int     Lq = (int)p.Lq - shift, tiles_end = skip == (int)p.Lq ? from : (Lq + QT - 1) / QT;
	const int64_t q_offset = p.q_offset + shift;
	const int last = (int)((int64_t)(split + 1) * a.part < n ? (int64_t)(split + 1) * a.part : n);
	const typename TK::reader at_q_(lane);
	const typename TV::reader at_g_(lane);
	carrier<T, DP, QT, S::NT>    pq[2];
	carrier<T, S::DV, QT, S::NT> pg;
	pq[0].begin(p.q_stride[2], a.columns);
	pg.begin(a.g.grad_out_stride[2], a.v_columns);
	row_stats<T, QT> rs;
	const T* const qb = static_cast<const T*>(p.q) + b * p.q_stride[0] + 2 * hk * G * p.q_stride[1] + shift * p.q_stride[2];
	const T* const gb = static_cast<const T*>(a.g.grad_out) + b * a.g.grad_out_stride[0] + hk * G * a.g.grad_out_stride[1] + shift * a.g.grad_out_stride[2];
	auto fetch = [&](int head, int at) {
		const T* const q = qb + 2 * head * p.q_stride[1];
		pq[0].load(q, at * QT, Lq), pq[1].load(q + p.q_stride[1], at * QT, Lq, pq[0]), pg.load(gb + head * a.g.grad_out_stride[1], at * QT, Lq);
		rs.load(a, b * p.H + hk * G + head, at * QT, shift, Lq);
	};
	int head = (int)((int64_t)split * a.part) / q_tiles, at = (int)((int64_t)split * a.part) - head * q_tiles;
	if(at < from) at = from;
	if(at >= tiles_end) head++, at = from;
	int buffer = 0;
	// (a workgroup none of whose keys counts has nothing to read)
	bool more = first != NONE && from < tiles_end && head * q_tiles + at < last;
	if(more) fetch(head, at);
	while(more) {
		unsigned char* const qs = smem + buffer * S::SET;
		unsigned char* const gs = qs + 2 * S::QTILE;
		float* const         st = reinterpret_cast<float*>(gs + S::GTILE);
		const int            q0 = at * QT, left = Lq - q0;
		const float          lam = lam_of(p, hk * G + head);
		if constexpr(S::BUFFERS == 1) __syncthreads();
		pq[0].store(qs, left >= QT, [&](int r) { return r < left; });
		pq[1].store(qs + S::QTILE, left >= QT, [&](int r) { return r < left; }, a.columns);
		pg.store(gs, left >= QT, [&](int r) { return r < left; });
		rs.store(st, a.factor);
		__syncthreads();
		if(++at == tiles_end) head++, at = from;
		more = head * q_tiles + at < last;
		if(more) fetch(head, at);
		const bool apart = rs.apart(st);
		float both[16];
		auto  add_values = [&](int row0) {
			const typename TV::reader at_g = S::PER_SIMD == 2 ? fresh(at_g_) : at_g_;
#pragma unroll
			for(int j = 0; j < TV::JOINTS; j++) {
				const u32x4 pf = kind<T>::pack(both + E * j);
#pragma unroll
				for(int db = 0; db < S::VBLOCKS; db++) dv[db] = kind<T>::mma(TV::col_frag(gs, row0, vblock0 + db, j, at_g), pf, dv[db]);
			}
		};
#pragma unroll 1
		for(int s = 0; s < S::SUB; s++) {
			const int row0 = 32 * (rwave * S::SUB + s);
			// the lane's rows need .. 15 of its 16 count
			const int  need = p.causal ? clamped(key - q_offset - (q0 + row0 + 16 * half)) : -64;
			const bool met = work && row0 < left && __any(in && need <= 15);
			if(met) {
				const bool diagonal = __any(in && need > 0);
				const typename TK::reader at_q = S::PER_SIMD == 2 ? fresh(at_q_) : at_q_;
				const typename TV::reader at_g = S::PER_SIMD == 2 ? fresh(at_g_) : at_g_;
				const float* const sm = st + row0 + 16 * half;
				f32x16 dp{};
#pragma unroll
				for(int i = 0; i < TV::STEPS; i++) dp = kind<T>::mma(TV::row_frag(gs, row0, i, at_g), vf[i], dp);
				// P1 - lam P2 (or the wavefront's part of it)
#pragma unroll
				for(int i = 0; i < MAPS; i++) {
					const int                  map = map0 + i;
					const unsigned char* const qm = qs + map * S::QTILE;
					f32x16 acc{};
#pragma unroll
					for(int k = 0; k < TK::STEPS; k++) acc = kind<T>::mma(TK::row_frag(qm, row0, k, at_q), kf[i][k], acc);
					float x[16];
					if(apart) {
						const f32x16 m = rs.sixteen(sm + (MOST + map) * QT), inv = rs.sixteen(sm + (INVERSE + map) * QT);
#pragma unroll
						for(int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_exp2f((acc[r] - m[r]) * a.factor) * inv[r];
					} else {
						const f32x16 taken = rs.sixteen(sm + (TAKEN + map) * QT);
#pragma unroll
						for(int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[r], a.factor, -taken[r]));
					}
					if(diagonal) {
#pragma unroll
						for(int r = 0; r < 16; r++) x[r] = r >= need ? x[r] : 0.f;
					}
					if(map == 1) {
#pragma unroll
						for(int r = 0; r < 16; r++) x[r] *= -lam;
					}
#pragma unroll
					for(int r = 0; r < 16; r++) both[r] = i == 0 ? x[r] : both[r] + x[r];
					const f32x16 less = rs.sixteen(sm + (LESS + map) * QT);
#pragma unroll
					for(int r = 0; r < 16; r++) x[r] *= dp[r] - less[r];
#pragma unroll
					for(int j = 0; j < TK::JOINTS; j++) {
						const u32x4 df = kind<T>::pack(x + E * j);
#pragma unroll
						for(int db = 0; db < TK::BLOCKS; db++) dk[i][db] = kind<T>::mma(TK::col_frag(qm, row0, db, j, at_q), df, dk[i][db]);
					}
				}
				if constexpr(MAPS == 2) add_values(row0);
			}
			if constexpr(MAPS == 1) {
				f32x4* const exchange = reinterpret_cast<f32x4*>(smem + S::BUFFERS * S::SET) + 256 * S::W * s + lane;
				if(met) {
#pragma unroll
					for(int i = 0; i < 4; i++) exchange[64 * (4 * wave + i)] = f32x4{both[4 * i], both[4 * i + 1], both[4 * i + 2], both[4 * i + 3]};
				}
				__syncthreads();
				if(met) {   // (and so it is for the other one, which has the same keys)
#pragma unroll
					for(int i = 0; i < 4; i++) {
						const f32x4 other = exchange[64 * (4 * (wave ^ 1) + i)];
#pragma unroll
						for(int e = 0; e < 4; e++) both[4 * i + e] += other[e];
					}
					add_values(row0);
				}
			}
		}
		if constexpr(S::BUFFERS == 2) buffer ^= 1;
	}
	float* const tables = reinterpret_cast<float*>(smem);
	if constexpr(RW > 1) {
#pragma unroll
		for(int i = 0; i < MAPS; i++) add_up<DP, RW>(tables + (MAPS == 2 ? group : 2 * group + map0) * RW * 32 * (DP + 4), rwave, lane, dk[i]);
	}
	if constexpr(RW > 1) add_up<S::DV, RW>(tables + group * RW * 32 * (S::DV + 4), rwave, lane, dv);
	if(!in) return;
	const int     D = (int)p.D, Dv = (int)p.Dv;
	const int64_t n_keys = p.B * p.Hkv * p.Lk, place = (b * p.Hkv + hk) * p.Lk + key;
	float* const  partial = a.partial + (int64_t)split * n_keys * (2 * D + Dv);
#pragma unroll
	for(int i = 0; i < MAPS; i++) {
		const int64_t to = (b * 2 * p.Hkv + 2 * hk + map0 + i) * p.Lk + key;
#pragma unroll
		for(int db = 0; db < TK::BLOCKS; db++) {
			if(db % RW != rwave) continue;
			float k[16];
#pragma unroll
			for(int r = 0; r < 16; r++) k[r] = lives ? dk[i][db][r] * p.softmax_scale : 0.f;
			if(a.splits > 1) store_columns(partial + to * D, 32 * db + 16 * half, D, k);
			else if(a.g.grad_k) store_columns(static_cast<T*>(a.g.grad_k) + to * D, 32 * db + 16 * half, D, k);
		}
	}
#pragma unroll
	for(int db = 0; db < S::VBLOCKS; db++) {
		if(db % RW != rwave) continue;
		float v[16];
#pragma unroll
		for(int r = 0; r < 16; r++) v[r] = lives ? dv[db][r] : 0.f;
		const int column = 32 * (vblock0 + db) + 16 * half;
		if(a.splits > 1) store_columns(partial + 2 * n_keys * D + place * Dv, column, Dv, v);
		else if(a.g.grad_v) store_columns(static_cast<T*>(a.g.grad_v) + place * Dv, column, Dv, v);
	}
}

// dlam: a workgroup per head, over the batch and the queries; each thread's numbers in turn, then the threads' pairwise
constexpr int LAM_THREADS = 1024;
__global__ void __launch_bounds__(LAM_THREADS) diff_lam_kernel(grad_args a) {
	__shared__ double sums[LAM_THREADS];
	const af3_diff_attention_params& p = a.p;
	const int64_t h = blockIdx.x, n = p.B * p.Lq;
	double sum = 0.0;
#pragma unroll 4
	for(int64_t i = threadIdx.x; i < n; i += LAM_THREADS) {
		const int64_t b = i / p.Lq;
		const int64_t row = (b * p.H + h) * p.Lq + (i - b * p.Lq);
		float         d2 = a.d2[row];
		for(uint32_t k = 0; k < a.shorts; k++) d2 += a.short_of[k * (p.B * p.H * p.Lq) + row];
		sum += (double)d2;
	}
	sums[threadIdx.x] = sum;
	for(int k = LAM_THREADS / 2; k; k >>= 1) {
		__syncthreads();
		if((int)threadIdx.x < k) sums[threadIdx.x] += sums[threadIdx.x + k];
	}
	if(threadIdx.x) return;
	if(p.lam_dtype == AF3_F32) static_cast<float*>(a.g.grad_lam)[h] = (float)-sums[0];
	else static_cast<uint16_t*>(a.g.grad_lam)[h] = kind<uint16_t>::bits((float)-sums[0]);
}

// The parts' sums added in order, of up to three results at once (a result of one part was written where it belongs).
constexpr int RESULTS = 3;
struct parts {
	const float* partial[RESULTS];
	int64_t      step[RESULTS], n[RESULTS];   // elements from one part to the next, elements
	uint32_t     splits[RESULTS], blocks[RESULTS];
	void*        out[RESULTS];
};
template <typename T>
__global__ void __launch_bounds__(THREADS) diff_sum_kernel(parts a) {
	uint32_t block = blockIdx.x;
	int      which = 0;
	while(which < RESULTS - 1 && block >= a.blocks[which]) block -= a.blocks[which++];
	const int64_t  i = ((int64_t)block * THREADS + threadIdx.x) * 4, n = a.n[which], step = a.step[which];
	const uint32_t splits = a.splits[which];
	const float*   at = a.partial[which] + i;
	T* const       out = static_cast<T*>(a.out[which]) + i;
	if(i >= n) return;
	if(i + 4 <= n) {
		f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
		for(uint32_t s = 0; s < splits; s++, at += step) sum += *reinterpret_cast<const f32x4_any*>(at);
#pragma unroll
		for(int e = 0; e < 4; e++) out[e] = kind<T>::bits(sum[e]);
	} else {
		for(int e = 0; i + e < n; e++) {
			float x = 0.f;
			for(uint32_t s = 0; s < splits; s++) x += at[s * step + e];
			out[e] = kind<T>::bits(x);
		}
	}
}

// ---- host side -------------------------------------------------------------------------------------------------------------
int width(const af3_diff_attention_params& p);   // (diff_attention.hip)

struct cut {
	int      sharing;   // wavefronts that share 32 rows (dq) or keys (dK, dV)
	uint32_t tiles, splits;
	int64_t  part;
};
inline int64_t over(int64_t n, int64_t per) { return (n + per - 1) / per; }
// bytes of a row of K as the kernels have it
int row_bytes(const af3_diff_attention_params& p) { return width(p) * (p.dtype == AF3_F32 ? 4 : 2); }
// the part of all (query, key) pairs that counts
double counting(const af3_diff_attention_params& p) {
	if(!p.causal) return 1.0;
	const double first = (double)p.q_offset + 1.0, last = (double)p.q_offset + (double)p.Lq, Lk = (double)p.Lk;   // keys of the first and the last query
	const double a = first < 0.0 ? 0.0 : first > Lk ? Lk : first, b = last < 0.0 ? 0.0 : last > Lk ? Lk : last;
	const double rising = b - a, full = last > Lk ? last - (first > Lk ? first : Lk) : 0.0;
	const double pairs = rising * (a + b) * 0.5 + full * Lk;
	return pairs <= 0.0 ? 1e-3 : pairs / ((double)p.Lq * Lk);
}
// `length` rows that results belong to, `alone` of them per workgroup where every wavefront has its own; `steps(sharing)` tiles of the other axis, of which a launch walks the part
// `counts`, the workgroups with the most first; `slots` workgroups fit the chip at a time; a tile costs load_us and block_us for each block of 32 x 32 that a wavefront has of it.
// Sharing makes more and shorter workgroups, so do parts of the long axis, whose results go through memory and are joined: whatever ends first.
template <typename U, typename F>
cut cut_for(int64_t length, int64_t groups, int64_t alone, int bytes, double counts, int64_t slots, double load_us, U block_us, double part_bytes, F steps) {
	constexpr double JOIN_US = 6.0, BYTES_PER_US = 2e6;
	const double tail = counts < 1.0 && by_tile(groups) ? 0.5 : 0.8;   // of the longest, behind all of them dealt out evenly
	// (8 x 16 x 768 x 64 causal, dQ: 117 us with 0.8 for both, 90.  Forward and all gradients with 0.8 and with 0.5, n causal pairs x length x 64: 8 x 1491 175 and 147; 16 x 768 126 and 121, x 1491 223 and
	// 232; 48 x 400 95 and 115, x 1024 195 and 189, x 1491 350 and 327; 128 x 400 136 and 155, x 768 307 and 266, x 1491 760 both.  Not causal: no difference in 20 sizes.)
	cut    best{};
	double best_us = 0.0;
	for(int sharing = 1; sharing <= (bytes > 128 ? 1 : 4); sharing *= 2) {
		const int64_t tiles = over(length, alone / sharing), n = steps(sharing), workgroups = groups * tiles;
		const double  tile_us = load_us * tile_rows(bytes, sharing) / 64 + block_us(sharing) * tile_rows(bytes, sharing) / (32 * sharing);
		for(int64_t parts = 1; parts <= 64 && (parts == 1 || 2 * parts <= n + 1); parts++) {
			const double longest = (double)over(n, parts), all = (double)workgroups * n * counts / slots;
			if(workgroups * parts > 0x7fffff && (sharing > 1 || parts > 1)) break;   // (times 512 threads inside 32 bits: so are those of the first choice, by what validate_diff_attention takes)
			const double us = (workgroups * parts <= slots ? longest : longest > all + tail * longest ? longest : all + tail * longest) * tile_us + (parts > 1 ? JOIN_US + parts * 2.0 * part_bytes / BYTES_PER_US : 0.0);
			if(best_us == 0.0 || us < best_us) best_us = us, best.sharing = sharing, best.tiles = (uint32_t)tiles, best.part = over(n, parts), best.splits = (uint32_t)over(n, best.part);
		}
	}
	return best;
}
cut dq_cut(const af3_diff_attention_params& p) {
	const int bytes = row_bytes(p);
	cut c = cut_for(p.H / p.Hkv * p.Lq, p.B * p.Hkv, 32 * DQ_THREADS / 64 * dq_maps(bytes) / 2, bytes, counting(p), 256, 0.4 + 0.009 * bytes, [&](int) { return (0.4 + 0.009 * bytes) * (p.dtype == AF3_F32 ? 2.0 : 1.0); },
					8.0 * p.B * p.H * p.Lq * p.D, [&](int sharing) { return over(p.Lk, tile_rows(bytes, sharing)); });
	c.part *= tile_rows(bytes, c.sharing);
	return c;
}
cut dkv_cut(const af3_diff_attention_params& p) {
	const int bytes = row_bytes(p);
	return cut_for(p.Lk, p.B * p.Hkv, bytes > 128 ? 64 : 128, bytes, counting(p), bytes > 64 ? 256 : 512, 0.3 + 0.006 * bytes, [&](int sharing) { return (0.5 + 0.009 * bytes) * (p.dtype == AF3_F32 ? 2.0 : sharing == 1 && bytes == 128 ? 0.7 : 1.0); },
				   4.0 * p.B * p.Hkv * p.Lk * (2 * p.D + p.Dv), [&](int sharing) { return p.H / p.Hkv * over(p.Lq, tile_rows(bytes, sharing)); });
}

int64_t packed_grad_bytes(const af3_diff_attention_params& p) {
	packing     k(p.dtype == AF3_F32 ? 4 : 2);
	const void* grad = nullptr;
	int64_t     stride[3] = {0, 0, 0};
	k.add(grad, stride, p.B, p.H, p.Lq, p.Dv, nullptr);
	return k.bytes;
}
struct grad_space {
	int64_t delta, shorts, dq, dkv, packed, bytes;   // floats; bytes of what is laid out anew, of all
};
grad_space grad_workspace(const af3_diff_attention_params& p) {
	const cut  q = dq_cut(p), kv = dkv_cut(p);
	grad_space w;
	w.delta = over(p.B * p.H * p.Lq, 4) * 4;
	w.shorts = over((int64_t)q.splits * q.sharing * p.B * p.H * p.Lq, 4) * 4;
	w.dq    = q.splits > 1 ? over(2 * (int64_t)q.splits * p.B * p.H * p.Lq * p.D, 4) * 4 : 0;
	w.dkv   = kv.splits > 1 ? over((int64_t)kv.splits * p.B * p.Hkv * p.Lk * (2 * p.D + p.Dv), 4) * 4 : 0;
	w.packed = packed_bytes(p) + packed_grad_bytes(p);
	w.bytes = w.packed + (2 * w.delta + w.shorts + w.dq + w.dkv) * 4;
	return w;
}

template <typename S, typename K>
int launch(K kernel, uint32_t grid, const grad_args& a, hipStream_t s) {
	constexpr int lds = S::LDS;
	if(lds > 65536 - 8192 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
		(void)hipGetLastError();
		return AF3_ERR_LAUNCH;
	}
	hipLaunchKernelGGL(kernel, dim3(grid), dim3(S::NT), lds, s, a);
	return launch_status();
}

template <typename T, int DP>
int backward(grad_args a, hipStream_t s) {
	const af3_diff_attention_params& p = a.p;
	const int64_t n_rows = 2 * p.B * p.H * p.Lq, n_keys = p.B * p.Hkv * p.Lk;
	constexpr bool SHARES = DP * (int)sizeof(T) <= 128;   // (wider rows: tiles that several wavefronts share leave neither registers nor LDS)
	parts    sums{};
	int      n_sums = 0;
	uint32_t sum_blocks = 0;
	auto add = [&](const float* partial, int64_t step, uint32_t splits, void* out, int64_t n) {
		if(!out) return;
		sums.partial[n_sums] = partial, sums.step[n_sums] = step, sums.n[n_sums] = n, sums.splits[n_sums] = splits, sums.out[n_sums] = out;
		sum_blocks += sums.blocks[n_sums] = (uint32_t)over(n, 4 * THREADS);
		n_sums++;
	};
	hipLaunchKernelGGL(diff_delta_kernel<T>, grid_of(over(p.B * p.H * p.Lq, THREADS / delta_lanes(p))), dim3(THREADS), 0, s, a);
	int rc = launch_status();
	if(rc != AF3_OK) return rc;
	if(!a.g.grad_lam) a.short_of = nullptr;
	if(a.g.grad_q || a.short_of) {
		const cut c = dq_cut(p);
		a.shorts = c.splits * c.sharing;
		a.tiles = c.tiles, a.splits = c.splits, a.part = c.part, a.partial = a.dq_space;
		const uint32_t grid = (uint32_t)(p.B * p.Hkv) * a.tiles * a.splits;
		rc = AF3_ERR_LAUNCH;
		if constexpr(SHARES) {
			if(c.sharing == 2) rc = launch<dq_shape<T, DP, 2>>(diff_dq_kernel<T, DP, 2>, grid, a, s);
			if(c.sharing == 4) rc = launch<dq_shape<T, DP, 4>>(diff_dq_kernel<T, DP, 4>, grid, a, s);
		}
		if(c.sharing == 1) rc = launch<dq_shape<T, DP, 1>>(diff_dq_kernel<T, DP, 1>, grid, a, s);
		if(rc != AF3_OK) return rc;
		if(a.splits > 1) add(a.partial, n_rows * p.D, c.splits, a.g.grad_q, n_rows * p.D);
	}
	if(a.g.grad_k || a.g.grad_v) {
		const cut c = dkv_cut(p);
		a.tiles = c.tiles, a.splits = c.splits, a.part = c.part, a.partial = a.dkv_space;
		const uint32_t grid = (uint32_t)(p.B * p.Hkv) * c.tiles * c.splits;
		rc = AF3_ERR_LAUNCH;
		if constexpr(SHARES) {
			if(c.sharing == 2) rc = launch<dkv_shape<T, DP, 2>>(diff_dkv_kernel<T, DP, 2>, grid, a, s);
			if(c.sharing == 4) rc = launch<dkv_shape<T, DP, 4>>(diff_dkv_kernel<T, DP, 4>, grid, a, s);
		}
		if(c.sharing == 1) rc = launch<dkv_shape<T, DP, 1>>(diff_dkv_kernel<T, DP, 1>, grid, a, s);
		if(rc != AF3_OK) return rc;
		if(c.splits > 1) {
			const int64_t step = n_keys * (2 * p.D + p.Dv);
			add(a.partial, step, c.splits, a.g.grad_k, 2 * n_keys * p.D);
			add(a.partial + 2 * n_keys * p.D, step, c.splits, a.g.grad_v, n_keys * p.Dv);
		}
	}
	if(n_sums) {
		hipLaunchKernelGGL(diff_sum_kernel<T>, dim3(sum_blocks), dim3(THREADS), 0, s, sums);
		if(rc = launch_status(); rc != AF3_OK) return rc;
	}
	if(a.g.grad_lam) {
		hipLaunchKernelGGL(diff_lam_kernel, dim3((uint32_t)p.H), dim3(LAM_THREADS), 0, s, a);
		return launch_status();
	}
	return AF3_OK;
}

int validate_grads(const af3_diff_attention_params* p, const af3_diff_attention_grads* g) {
	if(const int rc = validate_diff_attention(p); rc != AF3_OK) return rc;
	if(!g || !g->grad_out || !p->stats || (!g->grad_q && !g->grad_k && !g->grad_v && !g->grad_lam)) return AF3_ERR_NULL_POINTER;
	for(int i = 0; i < 3; i++)
		if(g->grad_out_stride[i] < 0) return AF3_ERR_BAD_STRIDE;
	const int bytes = p->dtype == AF3_F32 ? 4 : 2;
	if(p->Dv * bytes % 16 == 0 && p->Lq > 1 && !takes(p->Dv, g->grad_out_stride[2], bytes)) return AF3_ERR_BAD_STRIDE;   // (the workspace has no place for it)
	return AF3_OK;
}

}  // namespace diff
}  // namespace af3

using namespace af3;

extern "C" int64_t af3_diff_attention_backward_workspace_bytes(const af3_diff_attention_params* params) {
	if(const int rc = validate_diff_attention(params); rc != AF3_OK) return rc;
	return diff_gradients_fit(*params) ? diff::grad_workspace(*params).bytes : AF3_ERR_BAD_SHAPE;
}

extern "C" int af3_diff_attention_backward(const af3_diff_attention_params* params, const af3_diff_attention_grads* grads, void* hip_stream) {
	if(const int rc = diff::validate_grads(params, grads); rc != AF3_OK) return rc;
	const diff::grad_space w = diff::grad_workspace(*params);
	if(!grads->workspace || grads->workspace_bytes < w.bytes || (reinterpret_cast<uintptr_t>(grads->workspace) & 15)) return AF3_ERR_BAD_ARGUMENT;
	if(const int dc = current_device_status(); dc != AF3_OK) return dc;
	diff::grad_args a;
	a.p = *params, a.g = *grads, a.tiles = a.splits = 1, a.part = 0, a.partial = nullptr;
	a.factor = params->softmax_scale * LOG2E;
	diff::packing pack = diff::pack_inputs(a.p, a.columns, a.v_columns, grads->workspace);
	pack.add(a.g.grad_out, a.g.grad_out_stride, params->B, params->H, params->Lq, params->Dv, grads->workspace);
	a.d1 = reinterpret_cast<float*>(static_cast<unsigned char*>(grads->workspace) + w.packed), a.d2 = a.d1 + w.delta, a.short_of = a.d2 + w.delta, a.shorts = 0;
	a.dq_space = a.short_of + w.shorts, a.dkv_space = a.dq_space + w.dq;
	const hipStream_t s = static_cast<hipStream_t>(hip_stream);
	if(const int rc = pack.launch(s); rc != AF3_OK) return rc;
	const int wide = diff::width(*params);
	if(params->dtype == AF3_F32) return wide == 32 ? diff::backward<float, 32>(a, s) : diff::backward<float, 64>(a, s);
	return wide == 32 ? diff::backward<uint16_t, 32>(a, s) : wide == 64 ? diff::backward<uint16_t, 64>(a, s) : diff::backward<uint16_t, 128>(a, s);
}
