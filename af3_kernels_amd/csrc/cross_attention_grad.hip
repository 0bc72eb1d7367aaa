// The gradients of cross_attention.hip's attention: from P = softmax(S), out = P.V and dO = the gradient of out,
//     dV = P^T . dO,  dP = dO . V^T,  delta = rowsum(dO * out),  dS = P * (dP - delta),
//     dQ = scale dS . K,  dK = scale dS^T . Q,  dbias = dS summed over the batch.
// S and P are computed again from q, k and the two numbers per row that the forward pass left (maximum and 1 / sum: kept apart, since
// a maximum of the lowest float plus the logarithm of a sum is that maximum again).  Three kernels, none with atomics: each element
// of a result is summed by one workgroup, or by one per part of the long axis and a joining kernel, always in the same order.
//   cross_dq_kernel    32 query rows per wavefront, keys in tiles (writes delta too, and for a bias what it misses)
//   cross_dkv_kernel   32 keys per wavefront, query rows in tiles, over all query heads of the key head
//   cross_dbias_kernel 32 query rows x 32 keys per wavefront, over the batch
#include "cross_tiles.hpp"

#include <math.h>

namespace af3 {

int  validate_cross_attention(const af3_cross_attention_params* p);
bool cross_gradients_fit(const af3_cross_attention_params& p);

namespace cross {

struct grad_args {
	af3_cross_attention_params p;
	af3_cross_attention_grads  g;
	uint32_t tiles, splits;   // workgroups per (batch, key head), parts of the long axis
	int64_t  part;            // dq: keys per part; dkv: tiles of query rows per part
	float    factor;
	int32_t  whole;
	float*   delta;           // [B, H, Lq]
	float*   partial;         // dq: [splits][B H Lq][D]; dkv: [splits][2][B Hkv Lk][D]
	float *  dq_space, *dkv_space;
	float *  more, *row_sums; // what delta is short of, [B, H, Lq], or null; where cross_dq_kernel writes it: there, or its parts [splits][B, H, Lq]
};

// the sum of the wavefronts' results of equal shape, wavefront w keeps the blocks of columns that are w modulo N; `mine`: N tables of 32 x (DP + 4)
template <int DP, int N>
__device__ __forceinline__ void add_up(float* tables, int w, int lane, f32x16 (&o)[DP / 32]) {
	const int at = (lane & 31) * (DP + 4) + 16 * (lane >> 5);
#pragma unroll
	for(int db = 0; db < DP / 32; db++)
#pragma unroll
		for(int i = 0; i < 4; i++) *reinterpret_cast<f32x4*>(tables + w * 32 * (DP + 4) + at + 32 * db + 4 * i) = f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
	__syncthreads();
#pragma unroll
	for(int db = 0; db < DP / 32; db++) {
		if(db % N != w) continue;
		o[db] = f32x16{};
#pragma unroll
		for(int k = 0; k < N; k++)
#pragma unroll
			for(int i = 0; i < 4; i++) {
				const f32x4 v = *reinterpret_cast<const f32x4*>(tables + k * 32 * (DP + 4) + at + 32 * db + 4 * i);
#pragma unroll
				for(int e = 0; e < 4; e++) o[db][4 * i + e] += v[e];
			}
	}
}

// delta of a lane's query row from the lane's half of the gradient of out; the other half-wave has the other half
template <typename T, int DP, int N>
__device__ __forceinline__ float row_delta(const grad_args& a, const u32x4 (&gf)[N], int64_t b, int64_t h, int64_t qi, bool ok, int lane) {
	const af3_cross_attention_params& p = a.p;
	float delta = 0.f;
	u32x4 of[N];
	auto  add = [&] {
#pragma unroll
		for(int s = 0; s < N; s++)
#pragma unroll
			for(int e = 0; e < kind<T>::E; e++) delta = __builtin_fmaf(kind<T>::at(gf[s], e), kind<T>::at(of[s], e), delta);
	};
	load_operand<T, DP>(of, static_cast<const T*>(p.out) + b * p.out_stride[0] + h * p.out_stride[1] + qi * p.out_stride[2], ok, (int)p.D, lane);
	add();
	if(sizeof(T) == 2 && p.out_residual) {
		load_operand<T, DP>(of, static_cast<const T*>(p.out_residual) + ((b * p.H + h) * p.Lq + qi) * p.D, ok, (int)p.D, lane);
		add();
	}
	return sum_of_halves(delta);
}

// ---- dQ ----
template <typename T, int DP, int KW>
struct dq_shape {
	static constexpr int KT = KW == 4 ? 128 : 64, SUB = KT / (32 * KW), ROWS = 32 * (WAVES / KW);
	static constexpr int TILE = KT * tile<T, DP>::STRIDE;
	static constexpr int BUFFERS = 4 * TILE <= 81920 ? 2 : 1;
	static constexpr int JOIN = KW > 1 ? WAVES * 32 * (DP + 4) * 4 : 0;
	static constexpr int LDS = 2 * BUFFERS * TILE > JOIN ? 2 * BUFFERS * TILE : JOIN;
	static constexpr int REGISTERS = 8 * tile<T, DP>::STEPS + DP / 2 + 8 * passage<T, DP, KT>::N - (sizeof(T) == 2 ? 24 : 8);
};

template <typename T, int DP, int KW, bool BIAS>
__global__ void __launch_bounds__(THREADS, wavefronts(dq_shape<T, DP, KW>::REGISTERS + (BIAS && DP < 128 ? 32 : 0))) cross_dq_kernel(grad_args a) {
	using S  = dq_shape<T, DP, KW>;
	using TL = tile<T, DP>;
	constexpr int E = kind<T>::E, KT = S::KT;
	const af3_cross_attention_params& p = a.p;
	extern __shared__ __align__(16) unsigned char smem[];
	__shared__ live_keys<KT> live;

	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
	const int kwave = wave % KW, rwave = wave / KW;
	const share    own((uint32_t)blockIdx.x, (uint32_t)(p.B * p.Hkv), a.tiles * a.splits);
	const uint32_t split = own.piece / a.tiles, row_tile = own.piece - split * a.tiles;
	const int64_t  b = own.pair / (uint32_t)p.Hkv, hk = own.pair - (uint32_t)b * (uint32_t)p.Hkv;
	const int64_t G = p.H / p.Hkv, rows = G * p.Lq;
	const int     D = (int)p.D;

	const int64_t R  = (int64_t)row_tile * S::ROWS + 32 * rwave + (lane & 31);
	const bool    ok = R < rows;
	const int64_t g = ok ? R / p.Lq : 0, qi = ok ? R - g * p.Lq : 0, h = hk * G + g, row = (b * p.H + h) * p.Lq + qi;
	u32x4 qf[TL::STEPS], gf[TL::STEPS];
	load_operand<T, DP>(qf, static_cast<const T*>(p.q) + b * p.q_stride[0] + h * p.q_stride[1] + qi * p.q_stride[2], ok, D, lane);
	load_operand<T, DP>(gf, static_cast<const T*>(a.g.grad_out) + b * a.g.grad_out_stride[0] + h * a.g.grad_out_stride[1] + qi * a.g.grad_out_stride[2], ok, D, lane);
	const float delta = row_delta<T, DP>(a, gf, b, h, qi, ok, lane);
	if(ok && half == 0 && kwave == 0 && split == 0) a.delta[row] = delta;
	const float  m = ok ? p.stats[2 * row] : 0.f, inv = ok ? p.stats[2 * row + 1] : 0.f;
	const bool   apart = sizeof(T) == 4 || DP > 96 || __any(is_far(m * a.factor));   // (a row far from zero: in the logits' own units; 128 columns: registers for one form)
	const float  taken = whole_reference(m, inv, a.factor);
	const T* const kb = static_cast<const T*>(p.k) + b * p.k_stride[0] + hk * p.k_stride[1];
	const T* const vb = static_cast<const T*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[1];
	const T* const bias = BIAS ? static_cast<const T*>(p.bias) + h * p.bias_stride[0] + qi * p.bias_stride[1] : nullptr;
	const uint8_t* const mask = p.key_mask ? p.key_mask + b * p.key_mask_stride_b : nullptr;

	// The sum of a row of dS, which is zero but for what delta misses: out is made of probabilities rounded to bf16.  The bias's gradient is told (a sum over rows of it,
	// as a table's gradient is one, is made of what is left of such sums: at 8 x 12 x 512 x 512 x 64 and 32 buckets it was off by 0.0021 without this and is by 0.0014,
	// its last rounding to bf16 alone; no time lost, 30.2 us before and after).
	constexpr bool SUMS = BIAS && sizeof(T) == 2;
	__shared__ float wave_sums[SUMS && KW > 1 ? WAVES : 1][32];
	float row_sum = 0.f;
	f32x16 dq[TL::BLOCKS];
#pragma unroll
	for(int db = 0; db < TL::BLOCKS; db++) dq[db] = f32x16{};

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
			const int following = live.next(t + 1);
			if constexpr(S::BUFFERS == 1) __syncthreads();
			// (V is only multiplied row by row, and dS of a dropped key is not looked at; K's rows are added up under weights of zero)
			pk.store(ks, bits.full(), [&](int r) { return bits.keeps(r); });
			pv.store(vs, true, [](int) { return true; });
			__syncthreads();
			if(following >= 0) {
				pk.load(first + (int64_t)following * KT, end);
				pv.load(first + (int64_t)following * KT, end);
				fetch_bias(coming, following);
			}
#pragma unroll
			for(int s = 0; s < S::SUB; s++) {
				const int      block = kwave * S::SUB + s;
				const uint32_t keep  = bits.of_block(block);
				if(keep == 0u) continue;
				f32x16 acc{}, dp{};
#pragma unroll
				for(int i = 0; i < TL::STEPS; i++) acc = kind<T>::mma(TL::row_frag(ks, 32 * block, i, at), qf[i], acc);
#pragma unroll
				for(int i = 0; i < TL::STEPS; i++) dp = kind<T>::mma(TL::row_frag(vs, 32 * block, i, at), gf[i], dp);
				float x[16];
				auto logit = [&](int r) { return BIAS ? __builtin_fmaf(acc[r], p.softmax_scale, kind<T>::at(bs[s][r / E], r % E)) : acc[r]; };
				if(apart) {
#pragma unroll
					for(int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_exp2f((logit(r) - m) * a.factor) * inv * (dp[r] - delta);
				} else {
#pragma unroll
					for(int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(logit(r), a.factor, -taken)) * (dp[r] - delta);
				}
				if(keep != ~0u) drop_keys(x, keep, 0.f);
				if constexpr(SUMS)
					if(a.row_sums) {
#pragma unroll
						for(int r = 0; r < 16; r++) row_sum += x[r];
					}
#pragma unroll
				for(int j = 0; j < TL::JOINTS; j++) {
					const u32x4 f = kind<T>::pack(x + E * j);
#pragma unroll
					for(int db = 0; db < TL::BLOCKS; db++) dq[db] = kind<T>::mma(TL::col_frag(ks, 32 * block, db, j, at), f, dq[db]);
				}
			}
			t = following;
			if constexpr(S::BUFFERS == 2) buffer ^= 1;
		}
	}
	if constexpr(SUMS) {
		row_sum = sum_of_halves(row_sum);
		if constexpr(KW > 1) wave_sums[wave][lane & 31] = row_sum;
	}
	if constexpr(KW > 1) {
		__syncthreads();
		add_up<DP, KW>(reinterpret_cast<float*>(smem) + rwave * KW * 32 * (DP + 4), kwave, lane, dq);
	}
	if(!ok) return;
	if constexpr(SUMS)
		if(a.row_sums && kwave == 0 && half == 0) {
			if constexpr(KW > 1) {
				row_sum = 0.f;
#pragma unroll
				for(int w = 0; w < KW; w++) row_sum += wave_sums[rwave * KW + w][lane & 31];
			}
			a.row_sums[split * (p.B * p.H * p.Lq) + row] = row_sum;
		}
	if(!a.g.grad_q) return;
#pragma unroll
	for(int db = 0; db < TL::BLOCKS; db++) {
		if(db % KW != kwave) continue;
		float v[16];
#pragma unroll
		for(int r = 0; r < 16; r++) v[r] = dq[db][r] * p.softmax_scale;
		if(a.splits > 1) store_row16(a.partial + (split * (p.B * p.H * p.Lq) + row) * D, 32 * db + 16 * half, D, v);
		else store_row16(static_cast<T*>(a.g.grad_q) + row * D, 32 * db + 16 * half, D, v);
	}
}

// delta alone, for calls that want no gradient of q or the bias: 32 rows per wavefront, added up as cross_dq_kernel does
template <typename T, int DP>
__global__ void __launch_bounds__(THREADS) cross_delta_kernel(grad_args a) {
	const af3_cross_attention_params& p = a.p;
	const int     lane = threadIdx.x & 63;
	const int64_t row = ((int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6)) * 32 + (lane & 31);
	const bool    ok = row < p.B * p.H * p.Lq;
	const int64_t qi = ok ? row % p.Lq : 0, h = ok ? row / p.Lq % p.H : 0, b = ok ? row / p.Lq / p.H : 0;
	u32x4 gf[tile<T, DP>::STEPS];
	load_operand<T, DP>(gf, static_cast<const T*>(a.g.grad_out) + b * a.g.grad_out_stride[0] + h * a.g.grad_out_stride[1] + qi * a.g.grad_out_stride[2], ok, (int)p.D, lane);
	const float delta = row_delta<T, DP>(a, gf, b, h, qi, ok, lane);
	if(ok && lane < 32) a.delta[row] = delta;
}

// What the kernels with query rows in tiles keep of each row of a tile in LDS: delta with its sign turned (it begins the sum of dP), and, for bf16, the whole reference;
// maximum and 1 / sum for fp32 and for tiles with a row far from zero.  Behind them a word that says whether there is one.
constexpr int ROW_STATS = 4;
template <typename T, int QT>
struct row_stats {
	float taken, less, m, inv;   // of one row, on its way
	__device__ __forceinline__ void load(const grad_args& a, int64_t bh, int64_t q0, const float* more = nullptr) {
		taken = less = m = inv = 0.f;
		if((int)threadIdx.x >= QT) return;
		const bool ok = q0 + threadIdx.x < a.p.Lq;
		if(ok) {
			const int64_t row = bh * a.p.Lq + q0 + threadIdx.x;
			m = a.p.stats[2 * row], inv = a.p.stats[2 * row + 1], less = -(more ? a.delta[row] + more[row] : a.delta[row]);
		}
	}
	__device__ __forceinline__ void store(float* st, float factor) const {
		if((int)threadIdx.x >= QT) return;
		st[QT + threadIdx.x] = less, st[2 * QT + threadIdx.x] = m, st[3 * QT + threadIdx.x] = inv;
		if constexpr(sizeof(T) == 2) {
			st[threadIdx.x] = whole_reference(m, inv, factor);
			const bool far = __any(is_far(m * factor));   // (of 64 rows: a tile of 128 has two such words)
			if((threadIdx.x & 63) == 0) reinterpret_cast<int*>(st + ROW_STATS * QT)[threadIdx.x >> 6] = far;
		}
	}
	// whether the rows' maxima and sums are to be taken apart
	static __device__ __forceinline__ bool apart(const float* st) {
		if constexpr(sizeof(T) == 4) return true;
		const int* const far = reinterpret_cast<const int*>(st + ROW_STATS * QT);
		return __builtin_amdgcn_readfirstlane(QT > 64 ? far[0] | far[1] : far[0]) != 0;
	}
	static __device__ __forceinline__ f32x16 sixteen(const float* at) {
		f32x16 v;
#pragma unroll
		for(int i = 0; i < 4; i++) {
			const f32x4 x = *reinterpret_cast<const f32x4*>(at + 4 * i);
			v[4 * i] = x[0], v[4 * i + 1] = x[1], v[4 * i + 2] = x[2], v[4 * i + 3] = x[3];
		}
		return v;
	}
};

// ---- dK, dV ----
// RW: wavefronts that share 32 keys and each take 32 rows of a tile of query rows (1: every wavefront has its own keys and takes the whole tile)
// A bias comes through LDS as well, read like the columns of dO: a lane's 16 values lie in one column, and taken from memory one by one they were two thirds of the
// kernel's time (8 x 12 x 512 x 512 x 64: 102 us with a bias, 29 without).
template <typename T, int DP, int RW, bool BIAS>
struct dkv_shape {
	static constexpr int QT = RW == 4 ? 128 : sizeof(T) == 2 ? 64 : 32, SUB = QT / (32 * RW), KEYS = 32 * (WAVES / RW);
	static constexpr int TILE = QT * tile<T, DP>::STRIDE, STATS = ROW_STATS * QT * 4 + 16, BIASES = BIAS ? QT * tile<T, KEYS>::STRIDE : 0, SET = 2 * TILE + BIASES + STATS;
	static constexpr int BUFFERS = 2 * SET <= 81920 ? 2 : 1;
	static constexpr int JOIN = RW > 1 ? WAVES * 32 * (DP + 4) * 4 : 0;
	static constexpr int LDS = BUFFERS * SET > JOIN ? BUFFERS * SET : JOIN;
	static constexpr int REGISTERS = 8 * tile<T, DP>::STEPS + DP + 8 * passage<T, DP, QT>::N + (BIAS ? 4 * passage<T, KEYS, QT>::N : 0);
};

template <typename T, int DP, int RW, bool BIAS>
__global__ void __launch_bounds__(THREADS, wavefronts(dkv_shape<T, DP, RW, BIAS>::REGISTERS)) cross_dkv_kernel(grad_args a) {
	using S  = dkv_shape<T, DP, RW, BIAS>;
	using TL = tile<T, DP>;
	using TB = tile<T, S::KEYS>;
	constexpr int E = kind<T>::E, QT = S::QT;
	const af3_cross_attention_params& p = a.p;
	extern __shared__ __align__(16) unsigned char smem[];

	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
	const int rwave = wave % RW, kwave = wave / RW;
	const share    own((uint32_t)blockIdx.x, (uint32_t)(p.B * p.Hkv), a.tiles * a.splits);
	const uint32_t split = own.piece / a.tiles, key_tile = own.piece - split * a.tiles;
	const int64_t  b = own.pair / (uint32_t)p.Hkv, hk = own.pair - (uint32_t)b * (uint32_t)p.Hkv;
	const int64_t G = p.H / p.Hkv;
	const int     D = (int)p.D;

	const int64_t key0 = (int64_t)key_tile * S::KEYS, key = key0 + 32 * kwave + tile_row(lane & 31);   // (the order in which the biases' columns come)
	const bool    in = key < p.Lk;
	const bool    dead = p.stats[2 * ((b * p.H + hk * G) * p.Lq)] == -INFINITY;   // no live key in the batch row: P is 1 / Lk for all keys, S none of its business
	const bool    lives = in && (!p.key_mask || p.key_mask[b * p.key_mask_stride_b + key] != 0);
	u32x4 kf[TL::STEPS], vf[TL::STEPS];
	load_operand<T, DP>(kf, static_cast<const T*>(p.k) + b * p.k_stride[0] + hk * p.k_stride[1] + (in ? key : 0) * p.k_stride[2], in, D, lane);
	load_operand<T, DP>(vf, static_cast<const T*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[1] + (in ? key : 0) * p.v_stride[2], in, D, lane);
	const bool work = __any(lives || (dead && in));   // (of this wavefront)

	f32x16 dk[TL::BLOCKS], dv[TL::BLOCKS];
#pragma unroll
	for(int db = 0; db < TL::BLOCKS; db++) dk[db] = f32x16{}, dv[db] = f32x16{};

	const int64_t q_tiles = (p.Lq + QT - 1) / QT, n = G * q_tiles;
	const int64_t last = (int64_t)(split + 1) * a.part < n ? (int64_t)(split + 1) * a.part : n;
	const typename TL::reader at(lane);
	passage<T, DP, QT> pq, pg;
	pq.begin(nullptr, p.q_stride[2], D, a.whole);
	pg.begin(nullptr, a.g.grad_out_stride[2], D, a.whole);
	const typename TB::reader at_bias(lane);
	passage<T, S::KEYS, QT>   pb;
	if constexpr(BIAS) {
		const int keys = p.Lk - key0 < S::KEYS ? (int)(p.Lk - key0) : S::KEYS;
		pb.begin(nullptr, p.bias_stride[1], keys, keys % E == 0);
	}
	row_stats<T, QT> rs;
	auto fetch = [&](int64_t it) {
		const int64_t h = hk * G + it / q_tiles, q0 = it % q_tiles * QT;
		if constexpr(BIAS) {
			pb.base = static_cast<const T*>(p.bias) + h * p.bias_stride[0] + key0;
			pb.load(q0, p.Lq);
		}
		pq.base = static_cast<const T*>(p.q) + b * p.q_stride[0] + h * p.q_stride[1];
		pg.base = static_cast<const T*>(a.g.grad_out) + b * a.g.grad_out_stride[0] + h * a.g.grad_out_stride[1];
		pq.load(q0, p.Lq);
		pg.load(q0, p.Lq);
		rs.load(a, b * p.H + h, q0);
	};
	int     buffer = 0;
	int64_t it = (int64_t)split * a.part;
	// (a workgroup none of whose keys counts has nothing to read)
	const bool any = __syncthreads_or(work);
	if(!any) it = last;
	if(it < last) fetch(it);
	for(; it < last; it++) {
		unsigned char* const qs = smem + buffer * S::SET;
		unsigned char* const gs = qs + S::TILE;
		unsigned char* const bt = gs + S::TILE;
		float* const         st = reinterpret_cast<float*>(bt + S::BIASES);
		const int64_t        q0 = it % q_tiles * QT;
		if constexpr(S::BUFFERS == 1) __syncthreads();
		const int64_t left = p.Lq - q0;
		pq.store(qs, left >= QT, [&](int r) { return r < left; });
		pg.store(gs, left >= QT, [&](int r) { return r < left; });
		if constexpr(BIAS) pb.store(bt, left >= QT, [&](int r) { return r < left; });
		rs.store(st, a.factor);
		__syncthreads();
		const bool apart = rs.apart(st);
		if(it + 1 < last) fetch(it + 1);
		if(work) {
#pragma unroll
			for(int s = 0; s < S::SUB; s++) {
				const int row0 = 32 * (rwave * S::SUB + s);
				if(q0 + row0 >= p.Lq) continue;
				float x[16], y[16];
				const float* const sm = st + row0 + 16 * half;
				if(dead) {
#pragma unroll
					for(int r = 0; r < 16; r++) x[r] = sm[3 * QT + r], y[r] = 0.f;
				} else {
					f32x16 acc{}, dp = rs.sixteen(sm + QT);
#pragma unroll
					for(int i = 0; i < TL::STEPS; i++) acc = kind<T>::mma(TL::row_frag(qs, row0, i, at), kf[i], acc);
#pragma unroll
					for(int i = 0; i < TL::STEPS; i++) dp = kind<T>::mma(TL::row_frag(gs, row0, i, at), vf[i], dp);
					u32x4 bs[TB::JOINTS];
					if constexpr(BIAS) {
#pragma unroll
						for(int j = 0; j < TB::JOINTS; j++) bs[j] = TB::col_frag(bt, row0, kwave, j, at_bias);
					}
					auto logit = [&](int r) { return BIAS ? __builtin_fmaf(acc[r], p.softmax_scale, kind<T>::at(bs[r / E], r % E)) : acc[r]; };
					if(apart) {
						const f32x16 m = rs.sixteen(sm + 2 * QT), inv = rs.sixteen(sm + 3 * QT);
#pragma unroll
						for(int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_exp2f((logit(r) - m[r]) * a.factor) * inv[r];
					} else {
						const f32x16 taken = rs.sixteen(sm);
#pragma unroll
						for(int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(logit(r), a.factor, -taken[r]));
					}
#pragma unroll
					for(int r = 0; r < 16; r++) y[r] = x[r] * dp[r];
				}
#pragma unroll
				for(int j = 0; j < TL::JOINTS; j++) {
					const u32x4 pf = kind<T>::pack(x + E * j), df = kind<T>::pack(y + E * j);
#pragma unroll
					for(int db = 0; db < TL::BLOCKS; db++) {
						dv[db] = kind<T>::mma(TL::col_frag(gs, row0, db, j, at), pf, dv[db]);
						dk[db] = kind<T>::mma(TL::col_frag(qs, row0, db, j, at), df, dk[db]);
					}
				}
			}
		}
		if constexpr(S::BUFFERS == 2) buffer ^= 1;
	}
	if constexpr(RW > 1) {
		float* const tables = reinterpret_cast<float*>(smem) + kwave * RW * 32 * (DP + 4);
		__syncthreads();
		add_up<DP, RW>(tables, rwave, lane, dv);
		__syncthreads();
		add_up<DP, RW>(tables, rwave, lane, dk);
	}
	if(!in) return;
	const int64_t place = (b * p.Hkv + hk) * p.Lk + key, n_keys = p.B * p.Hkv * p.Lk;
	const bool    counts_v = lives || dead, counts_k = lives && !dead;
#pragma unroll
	for(int db = 0; db < TL::BLOCKS; db++) {
		if(db % RW != rwave) continue;
		float v[16], k[16];
#pragma unroll
		for(int r = 0; r < 16; r++) v[r] = counts_v ? dv[db][r] : 0.f, k[r] = counts_k ? dk[db][r] * p.softmax_scale : 0.f;
		if(a.splits > 1) {
			store_row16(a.partial + (2 * split * n_keys + place) * D, 32 * db + 16 * half, D, k);
			store_row16(a.partial + ((2 * split + 1) * n_keys + place) * D, 32 * db + 16 * half, D, v);
		} else {
			if(a.g.grad_k) store_row16(static_cast<T*>(a.g.grad_k) + place * D, 32 * db + 16 * half, D, k);
			if(a.g.grad_v) store_row16(static_cast<T*>(a.g.grad_v) + place * D, 32 * db + 16 * half, D, v);
		}
	}
}

// The parts' sums added in order, of up to four results at once (a result of one part was written where it belongs).
constexpr int RESULTS = 4;
struct parts {
	const float* partial[RESULTS];
	int64_t      step[RESULTS], n[RESULTS];   // elements from one part to the next, elements
	uint32_t     splits[RESULTS], blocks[RESULTS];
	void*        out[RESULTS];
	bool         wide[RESULTS];   // fp32, whatever T is
};
template <typename T>
__global__ void __launch_bounds__(THREADS) cross_sum_kernel(parts a) {
	uint32_t block = blockIdx.x;
	int      which = 0;
	while(which < RESULTS - 1 && block >= a.blocks[which]) block -= a.blocks[which++];
	const int64_t  i = ((int64_t)block * THREADS + threadIdx.x) * 4, n = a.n[which], step = a.step[which];
	const uint32_t splits = a.splits[which];
	const float*   at = a.partial[which] + i;
	T* const       out = static_cast<T*>(a.out[which]) + i;
	float* const   wide = a.wide[which] ? static_cast<float*>(a.out[which]) + i : nullptr;
	if(i >= n) return;
	if(i + 4 <= n) {
		f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
		for(uint32_t s = 0; s < splits; s++, at += step) sum += *reinterpret_cast<const f32x4_any*>(at);
#pragma unroll
		for(int e = 0; e < 4; e++)
			if(wide) wide[e] = sum[e];
			else out[e] = kind<T>::bits(sum[e]);
	} else {
		for(int e = 0; i + e < n; e++) {
			float x = 0.f;
			for(uint32_t s = 0; s < splits; s++) x += at[s * step + e];
			if(wide) wide[e] = x;
			else out[e] = kind<T>::bits(x);
		}
	}
}

// ---- dbias ----
// A workgroup has 64 query rows x 64 keys (a wavefront 32 x 32 of them) and goes through the batch; q, dO, k and v come as tiles.  Few sums to hold leave room for
// many wavefronts: 128 keys with K and V as operands straight from memory took 57 us at 8 x 12 x 512 x 512 x 64, where the loads of every batch row stood alone.  Nor are
// tiles fetched ahead of their use: the registers they would wait in cost the third workgroup of a compute unit, which hides more (ahead, two workgroups: 44.5 us there and
// 76 at 4 x 16 x 768 x 768 x 64; so, three: 29.8 and 49; ahead and three, with spills: 74).  fp32 stays at what it needs without spills.
template <typename T, int DP>
struct dbias_shape {
	static constexpr int QT = 64, KT = 64, TILE = 64 * tile<T, DP>::STRIDE, STATS = ROW_STATS * QT * 4 + 16, LDS = 4 * TILE + STATS;
	static constexpr int REGISTERS = (sizeof(T) == 2 ? 32 : 48) + 16 * passage<T, DP, 64>::N;
};

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, wavefronts(dbias_shape<T, DP>::REGISTERS)) cross_dbias_kernel(grad_args a) {
	using S  = dbias_shape<T, DP>;
	using TL = tile<T, DP>;
	constexpr int QT = S::QT, KT = S::KT, E = kind<T>::E;
	const af3_cross_attention_params& p = a.p;
	extern __shared__ __align__(16) unsigned char smem[];
	unsigned char *const qs = smem, *const gs = qs + S::TILE, *const ks = gs + S::TILE, *const vs = ks + S::TILE;
	float* const st = reinterpret_cast<float*>(vs + S::TILE);

	const int      lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
	const uint32_t key_tiles = (uint32_t)((p.Lk + KT - 1) / KT);
	const share    own((uint32_t)blockIdx.x, (uint32_t)p.H, a.tiles * key_tiles);
	const uint32_t q_tile = own.piece / key_tiles, key_tile = own.piece - q_tile * key_tiles;
	const int64_t  q0 = (int64_t)q_tile * QT, k0 = (int64_t)key_tile * KT, h = own.pair, hk = h / (p.H / p.Hkv);
	const int      row0 = 32 * (wave >> 1), col0 = 32 * (wave & 1);
	const int      D = (int)p.D;
	// (K and V as B operands are read like A operands: lane n holds key tile_row(n) of the block)
	const int64_t  key = k0 + col0 + tile_row(lane & 31);
	const bool     in = key < p.Lk;

	float sum[16];
	u32x4 bs[16 / E];
	{
		T entry[16];
#pragma unroll
		for(int r = 0; r < 16; r++) {
			const int64_t q = q0 + row0 + 16 * half + r;
			sum[r] = 0.f, entry[r] = T(0);
			if(in && q < p.Lq) entry[r] = static_cast<const T*>(p.bias)[h * p.bias_stride[0] + q * p.bias_stride[1] + key];
		}
#pragma unroll
		for(int i = 0; i < 16 / E; i++) __builtin_memcpy(&bs[i], entry + E * i, 16);
	}
	auto logit = [&](float qk, int r) { return __builtin_fmaf(qk, p.softmax_scale, kind<T>::at(bs[r / E], r % E)); };
	const typename TL::reader at(lane);
	passage<T, DP, 64> pq, pg, pk, pv;
	pq.begin(nullptr, p.q_stride[2], D, a.whole);
	pg.begin(nullptr, a.g.grad_out_stride[2], D, a.whole);
	pk.begin(nullptr, p.k_stride[2], D, a.whole);
	pv.begin(nullptr, p.v_stride[2], D, a.whole);
	row_stats<T, QT> rs;
	auto fetch = [&](int64_t b) {
		pq.base = static_cast<const T*>(p.q) + b * p.q_stride[0] + h * p.q_stride[1];
		pg.base = static_cast<const T*>(a.g.grad_out) + b * a.g.grad_out_stride[0] + h * a.g.grad_out_stride[1];
		pk.base = static_cast<const T*>(p.k) + b * p.k_stride[0] + hk * p.k_stride[1];
		pv.base = static_cast<const T*>(p.v) + b * p.v_stride[0] + hk * p.v_stride[1];
		pq.load(q0, p.Lq);
		pg.load(q0, p.Lq);
		pk.load(k0, p.Lk);
		pv.load(k0, p.Lk);
		rs.load(a, b * p.H + h, q0, a.more);
	};
	const int64_t rows_left = p.Lq - q0, keys_left = p.Lk - k0;
	// Workgroups begin with different batch rows: beginning alike, all of them waited for each row's way from memory, a row after the other.
	int64_t b = own.piece % p.B;
	for(int64_t left = p.B; left > 0; left--) {
		fetch(b);
		const bool lives = in && (!p.key_mask || p.key_mask[b * p.key_mask_stride_b + key] != 0);
		b = b + 1 < p.B ? b + 1 : 0;   // (the next one)
		__syncthreads();   // (nobody reads the batch row before any more)
		pq.store(qs, rows_left >= 64, [&](int r) { return r < rows_left; });
		pg.store(gs, rows_left >= 64, [&](int r) { return r < rows_left; });
		pk.store(ks, keys_left >= 64, [&](int r) { return r < keys_left; });
		pv.store(vs, keys_left >= 64, [&](int r) { return r < keys_left; });
		rs.store(st, a.factor);
		__syncthreads();
		if(st[2 * QT] == -INFINITY || !__any(lives)) continue;   // (-inf: a batch row without a live key)
		const float* const sm = st + row0 + 16 * half;
		f32x16 acc{}, dp = rs.sixteen(sm + QT);
#pragma unroll
		for(int i = 0; i < TL::STEPS; i++) acc = kind<T>::mma(TL::row_frag(qs, row0, i, at), TL::row_frag(ks, col0, i, at), acc);
#pragma unroll
		for(int i = 0; i < TL::STEPS; i++) dp = kind<T>::mma(TL::row_frag(gs, row0, i, at), TL::row_frag(vs, col0, i, at), dp);
		float x[16];
		if(rs.apart(st)) {
			const f32x16 m = rs.sixteen(sm + 2 * QT), inv = rs.sixteen(sm + 3 * QT);
#pragma unroll
			for(int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_exp2f((logit(acc[r], r) - m[r]) * a.factor) * inv[r];
		} else {
			const f32x16 taken = rs.sixteen(sm);
#pragma unroll
			for(int r = 0; r < 16; r++) x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(logit(acc[r], r), a.factor, -taken[r]));
		}
#pragma unroll
		for(int r = 0; r < 16; r++) sum[r] += lives ? x[r] * dp[r] : 0.f;   // (what k, v and bias hold at a dropped key stays in its own lane)
	}
	if(!in) return;
	T* const out = static_cast<T*>(a.g.grad_bias) + h * p.Lq * p.Lk + key;
#pragma unroll
	for(int r = 0; r < 16; r++) {
		const int64_t q = q0 + row0 + 16 * half + r;
		if(q < p.Lq) {
			const T rounded = kind<T>::bits(sum[r]);
			out[q * p.Lk] = rounded;
			if(sizeof(T) == 2 && a.g.grad_bias_residual) static_cast<T*>(a.g.grad_bias_residual)[(h * p.Lq + q) * p.Lk + key] = kind<T>::bits(sum[r] - kind<T>::value(rounded));
		}
	}
}

// ---- host side -------------------------------------------------------------------------------------------------------------
struct cut {
	bool     shared;   // wavefronts share 32 rows (dq) or keys (dkv)
	uint32_t tiles, splits;
	int64_t  part;
};
inline int64_t over(int64_t n, int64_t per) { return (n + per - 1) / per; }

// `length` rows that results belong to (128 or 32 of them per workgroup), `steps(shared)` tiles of the other axis.  Wavefronts share where the workgroups of 32 fit the chip
// together: dQ / dK and dV, us, alone and shared, at 2 x 8 x 384 x 1024 x 64 20.6, 14.2 / 17.6, 13.0, 1 x 8 x 1024 x 1024 x 64 25.8, 17.3 / 38.3, 19.6 (256 workgroups of 32),
// 8 x 12 x 512 x 512 x 64 25.0, 43.0 / 29.5, 43.8 (1536), fp32 2 x 8 x 259 x 384 x 32 25.3, 14.9 / 31.4, 15.8.
template <typename F>
cut cut_for(int64_t length, int64_t groups, bool may_share, int64_t slots, double tile_us, double part_bytes, F steps) {
	cut c;
	c.shared = may_share && (length <= 32 || over(length, 32) * groups <= 512);
	c.tiles  = (uint32_t)over(length, c.shared ? 32 : 128);
	const int64_t n = steps(c.shared);
	const int64_t sp = parts_for(groups * c.tiles, slots, n, tile_us * (c.shared ? 1.0 : 0.6), part_bytes, 64);
	c.part   = over(n, sp);
	c.splits = (uint32_t)over(n, c.part);
	return c;
}
cut dq_cut(const af3_cross_attention_params& p) {
	const bool fp32 = p.dtype == AF3_F32;
	cut c = cut_for(p.H / p.Hkv * p.Lq, p.B * p.Hkv, true, p.D > 64 || (fp32 && p.D > 32) ? 256 : 512, (0.5 + 0.016 * p.D) * (fp32 ? 3.0 : 1.0), 4.0 * p.B * p.H * p.Lq * p.D,
					[&](bool shared) { return over(p.Lk, shared ? 128 : 64); });
	c.part *= c.shared ? 128 : 64;
	return c;
}
cut dkv_cut(const af3_cross_attention_params& p) {
	// (fp32 beyond 64 columns: the tile of 128 rows leaves no registers for the sums)
	const bool fp32 = p.dtype == AF3_F32;
	return cut_for(p.Lk, p.B * p.Hkv, !fp32 || p.D <= 64, p.D > 64 || (fp32 && p.D > 32) ? 256 : 512, (0.6 + 0.022 * p.D) * (fp32 ? 3.0 : 1.0), 8.0 * p.B * p.Hkv * p.Lk * p.D,
				   [&](bool shared) { return p.H / p.Hkv * over(p.Lq, shared ? 128 : fp32 ? 32 : 64); });
}

struct grad_space {
	int64_t delta, more, row_sums, dq, dkv, bytes;   // floats
};
grad_space grad_workspace(const af3_cross_attention_params& p) {
	const cut  q = dq_cut(p), kv = dkv_cut(p);
	grad_space w;
	w.delta = over(p.B * p.H * p.Lq, 4) * 4;
	w.more  = p.bias && p.dtype == AF3_BF16 ? w.delta : 0;
	w.row_sums = w.more && q.splits > 1 ? over(q.splits * p.B * p.H * p.Lq, 4) * 4 : 0;
	w.dq    = q.splits > 1 ? over(q.splits * p.B * p.H * p.Lq * p.D, 4) * 4 : 0;
	w.dkv   = kv.splits > 1 ? 2 * (int64_t)kv.splits * p.B * p.Hkv * p.Lk * p.D : 0;
	w.bytes = (w.delta + w.more + w.row_sums + w.dq + w.dkv) * 4;
	return w;
}

template <typename K>
int launch(K kernel, int lds, uint32_t grid, const grad_args& a, hipStream_t s) {
	if(lds > 65536 - 8192 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
		(void)hipGetLastError();
		return AF3_ERR_LAUNCH;
	}
	hipLaunchKernelGGL(kernel, dim3(grid), dim3(THREADS), lds, s, a);
	return launch_status();
}

template <typename T, int DP>
int backward(grad_args a, hipStream_t s) {
	const af3_cross_attention_params& p = a.p;
	const int64_t n_rows = p.B * p.H * p.Lq, n_keys = p.B * p.Hkv * p.Lk;
	parts    sums{};
	int      n_sums = 0;
	uint32_t sum_blocks = 0;
	auto add = [&](const float* partial, int64_t step, uint32_t splits, void* out, int64_t n, bool wide = false) {
		if(!out) return;
		sums.wide[n_sums] = wide;
		sums.partial[n_sums] = partial, sums.step[n_sums] = step, sums.n[n_sums] = n, sums.splits[n_sums] = splits, sums.out[n_sums] = out;
		sum_blocks += sums.blocks[n_sums] = (uint32_t)over(n, 4 * THREADS);
		n_sums++;
	};
	if(!a.g.grad_bias) a.more = nullptr;
	if(a.g.grad_q || a.more) {
		const cut c = dq_cut(p);
		a.tiles = c.tiles, a.splits = c.splits, a.part = c.part, a.partial = a.dq_space;
		a.row_sums = a.more && c.splits > 1 ? a.row_sums : a.more;
		const uint32_t grid = (uint32_t)(p.B * p.Hkv) * c.tiles * c.splits;
		int rc;
		if(c.shared) rc = p.bias ? launch(cross_dq_kernel<T, DP, 4, true>, dq_shape<T, DP, 4>::LDS, grid, a, s) : launch(cross_dq_kernel<T, DP, 4, false>, dq_shape<T, DP, 4>::LDS, grid, a, s);
		else rc = p.bias ? launch(cross_dq_kernel<T, DP, 1, true>, dq_shape<T, DP, 1>::LDS, grid, a, s) : launch(cross_dq_kernel<T, DP, 1, false>, dq_shape<T, DP, 1>::LDS, grid, a, s);
		if(rc != AF3_OK) return rc;
		if(c.splits > 1) {
			add(a.partial, n_rows * p.D, c.splits, a.g.grad_q, n_rows * p.D);
			add(a.row_sums, n_rows, c.splits, a.more, n_rows, true);
		}
	} else {
		hipLaunchKernelGGL((cross_delta_kernel<T, DP>), dim3((uint32_t)over(n_rows, 32 * WAVES)), dim3(THREADS), 0, s, a);
		if(const int rc = launch_status(); rc != AF3_OK) return rc;
	}
	if(a.g.grad_k || a.g.grad_v) {
		const cut c = dkv_cut(p);
		a.tiles = c.tiles, a.splits = c.splits, a.part = c.part, a.partial = a.dkv_space;
		const uint32_t grid = (uint32_t)(p.B * p.Hkv) * c.tiles * c.splits;
		int rc = AF3_ERR_LAUNCH;
		if constexpr(sizeof(T) == 2 || DP <= 64)
			if(c.shared) rc = p.bias ? launch(cross_dkv_kernel<T, DP, 4, true>, dkv_shape<T, DP, 4, true>::LDS, grid, a, s) : launch(cross_dkv_kernel<T, DP, 4, false>, dkv_shape<T, DP, 4, false>::LDS, grid, a, s);
		if(!c.shared) rc = p.bias ? launch(cross_dkv_kernel<T, DP, 1, true>, dkv_shape<T, DP, 1, true>::LDS, grid, a, s) : launch(cross_dkv_kernel<T, DP, 1, false>, dkv_shape<T, DP, 1, false>::LDS, grid, a, s);
		if(rc != AF3_OK) return rc;
		if(c.splits > 1) {
			add(a.partial, 2 * n_keys * p.D, c.splits, a.g.grad_k, n_keys * p.D);
			add(a.partial + n_keys * p.D, 2 * n_keys * p.D, c.splits, a.g.grad_v, n_keys * p.D);
		}
	}
	if(n_sums) {
		hipLaunchKernelGGL(cross_sum_kernel<T>, dim3(sum_blocks), dim3(THREADS), 0, s, sums);
		if(const int rc = launch_status(); rc != AF3_OK) return rc;
	}
	if(a.g.grad_bias) {
		using S = dbias_shape<T, DP>;
		a.tiles = (uint32_t)over(p.Lq, S::QT);
		return launch(cross_dbias_kernel<T, DP>, S::LDS, (uint32_t)(p.H * a.tiles * over(p.Lk, S::KT)), a, s);
	}
	return AF3_OK;
}
template <typename T>
int backward_type(const grad_args& a, hipStream_t s) {
	if(a.p.D <= 32) return backward<T, 32>(a, s);
	if(a.p.D <= 64) return backward<T, 64>(a, s);
	if(a.p.D <= 96) return backward<T, 96>(a, s);
	return backward<T, 128>(a, s);
}

int validate_grads(const af3_cross_attention_params* p, const af3_cross_attention_grads* g) {
	if(const int rc = validate_cross_attention(p); rc != AF3_OK) return rc;
	if(!g || !g->grad_out || !p->stats || (!g->grad_q && !g->grad_k && !g->grad_v && !g->grad_bias)) return AF3_ERR_NULL_POINTER;
	if((g->grad_bias && !p->bias) || (g->grad_bias_residual && !g->grad_bias)) return AF3_ERR_NULL_POINTER;
	for(int i = 0; i < 3; i++)
		if(g->grad_out_stride[i] < 0) return AF3_ERR_BAD_STRIDE;
	if(g->grad_bias_residual && p->dtype != AF3_BF16) return AF3_ERR_BAD_DTYPE;   // (nothing would be written there)
	// (the bias's gradient: a workgroup for every 64 x 64 entries.  cross.py and host.cpp refuse such a call before its forward pass)
	if(!cross_gradients_fit(*p) || (g->grad_bias && p->H * over(p->Lq, 64) * over(p->Lk, 64) > 0xffffff)) return AF3_ERR_BAD_SHAPE;
	return AF3_OK;
}

}  // namespace cross
}  // namespace af3

using namespace af3;

extern "C" int64_t af3_cross_attention_backward_workspace_bytes(const af3_cross_attention_params* params) {
	if(const int rc = validate_cross_attention(params); rc != AF3_OK) return rc;
	return cross_gradients_fit(*params) ? cross::grad_workspace(*params).bytes : AF3_ERR_BAD_SHAPE;
}

extern "C" int af3_cross_attention_backward(const af3_cross_attention_params* params, const af3_cross_attention_grads* grads, void* hip_stream) {
	if(const int rc = cross::validate_grads(params, grads); rc != AF3_OK) return rc;
	const cross::grad_space w = cross::grad_workspace(*params);
	if(!grads->workspace || grads->workspace_bytes < w.bytes || (reinterpret_cast<uintptr_t>(grads->workspace) & 15)) return AF3_ERR_BAD_ARGUMENT;
	if(const int dc = current_device_status(); dc != AF3_OK) return dc;
	cross::grad_args a;
	a.p = *params, a.g = *grads, a.tiles = a.splits = 1, a.part = 0;
	a.factor  = params->bias ? LOG2E : params->softmax_scale * LOG2E;
	a.whole   = params->D * (params->dtype == AF3_F32 ? 4 : 2) % 16 == 0;
	a.delta   = static_cast<float*>(grads->workspace);
	a.more     = w.more ? a.delta + w.delta : nullptr;
	a.row_sums = a.delta + w.delta + w.more;
	a.partial  = nullptr, a.dq_space = a.row_sums + w.row_sums, a.dkv_space = a.dq_space + w.dq;
	const hipStream_t s = static_cast<hipStream_t>(hip_stream);
	return params->dtype == AF3_F32 ? cross::backward_type<float>(a, s) : cross::backward_type<uint16_t>(a, s);
}
