// The norms around a block with its gate and residual scale, and their gradients: for every row of C channels
//     z = post_norm(y) post_weight,   r = residual_scale x + act(gate) z,   h = norm(r) weight + bias.
// af3_residual_norm_forward / _backward.
//
// A row is read once, held in registers through its reductions (64 to 1024 threads to a row, 8 or 16 channels each) and written once: the forward pass is bound by its bytes, the gradient by its
// vector instructions and by what its rows wait for at the norms' sums.  The gradient works r out again from x, y and the gate, unrounded as the forward pass had it, with the two norms' statistics from there.  What many
// rows share (a weight by channel, a gate by sequence) has its gradient summed in registers over the rows of a workgroup; workgroups' sums are joined by a second kernel in
// a fixed order.
// 4 x 2048 rows of 4096 channels in bf16, all of it: 165 us for 109 that a copy of the same bytes takes, each read and written once (the gradient reads x and y again); the forward pass 49 of them,
// 268 MB, 5.5 TB/s, the gradient 107, 428 MB, 4.0 TB/s.  Rows of more than
// 8192 channels spill in the gradient's kernel, whose 1024 threads have 128 registers each.
#include "launch_grid.hpp"
#include "mfma_helpers.hpp"

// (products and sums are fused where fmaf says so: the kernels' instantiations then agree to the last bit, whichever gradients are wanted)
#pragma clang fp contract(off)

namespace af3 {
namespace rnorm {

constexpr int E = 8;   // channels side by side in a thread

template <typename T>
struct eight {   // 8 channels as they lie in memory
	T e[E];
	__device__ __forceinline__ void load(const T* p) {
		if constexpr(sizeof(T) == 2) {
			const u32x4_any v = *reinterpret_cast<const u32x4_any*>(p);
			__builtin_memcpy(e, &v, 16);
		} else {
			const f32x4_any v0 = *reinterpret_cast<const f32x4_any*>(p), v1 = *reinterpret_cast<const f32x4_any*>(p + 4);
			__builtin_memcpy(e, &v0, 16), __builtin_memcpy(e + 4, &v1, 16);
		}
	}
	__device__ __forceinline__ void store(T* p) const {
		if constexpr(sizeof(T) == 2) {
			u32x4_any v;
			__builtin_memcpy(&v, e, 16);
			*reinterpret_cast<u32x4_any*>(p) = v;
		} else {
			f32x4_any v0, v1;
			__builtin_memcpy(&v0, e, 16), __builtin_memcpy(&v1, e + 4, 16);
			*reinterpret_cast<f32x4_any*>(p) = v0, *reinterpret_cast<f32x4_any*>(p + 4) = v1;
		}
	}
};
__device__ __forceinline__ float value(uint16_t x) { return bf16_bits_to_f32(x); }
__device__ __forceinline__ float value(float x) { return x; }
template <typename T> __device__ __forceinline__ T bits(float x);
template <> __device__ __forceinline__ uint16_t bits<uint16_t>(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
template <> __device__ __forceinline__ float bits<float>(float x) { return x; }

// A row's channels over TPR threads: thread t has channels 8 t .. 8 t + 7 of every stretch of 8 TPR
template <typename T, int TPR, int NP>
struct row_of {
	int  c0, C;   // c0: of the first stretch
	__device__ __forceinline__ row_of(int lane, int C_) : c0(E * lane), C(C_) {}
	__device__ __forceinline__ int  at(int n) const { return c0 + E * TPR * n; }
	__device__ __forceinline__ bool whole(int n) const { return at(n) + E <= C; }
	__device__ __forceinline__ bool in(int n, int e) const { return at(n) + e < C; }
	__device__ __forceinline__ void load(eight<T> (&v)[NP], const T* row) const {
#pragma unroll
		for(int n = 0; n < NP; n++) {
			if(whole(n)) v[n].load(row + at(n));
			else {
#pragma unroll
				for(int e = 0; e < E; e++) {
					v[n].e[e] = T(0);
					if(in(n, e)) v[n].e[e] = row[at(n) + e];
				}
			}
		}
	}
	__device__ __forceinline__ void store(T* row, const float (&v)[NP][E]) const {
#pragma unroll
		for(int n = 0; n < NP; n++) {
			eight<T> o;
#pragma unroll
			for(int e = 0; e < E; e++) o.e[e] = bits<T>(v[n][e]);
			if(whole(n)) o.store(row + at(n));
			else {
#pragma unroll
				for(int e = 0; e < E; e++)
					if(in(n, e)) row[at(n) + e] = o.e[e];
			}
		}
	}
	__device__ __forceinline__ void store_sums(float* row, const float (&v)[NP][E]) const {
#pragma unroll
		for(int n = 0; n < NP; n++)
#pragma unroll
			for(int e = 0; e < E; e++)
				if(in(n, e)) row[at(n) + e] = v[n][e];
	}
};

template <int CTRL, int ROWS>
__device__ __forceinline__ float add_from(float x) {
	return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, ROWS, 0xf, true));
}
// the sum over a wavefront, in all lanes (rows of 16 lanes by shifts, then row by row; lane 63 has it)
__device__ __forceinline__ float wave_sum(float x) {
	x = add_from<0x111, 0xf>(x), x = add_from<0x112, 0xf>(x), x = add_from<0x114, 0xf>(x), x = add_from<0x118, 0xf>(x);
	x = add_from<0x142, 0xa>(x), x = add_from<0x143, 0xc>(x);
	return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
// Sums over the TPR threads of a row.  More than one wavefront: through LDS, places of a sum and the one after it differ, so that one barrier per sum is enough.
template <int TPR>
struct row_sums {
	float* lds;   // [2][TPR / 64][2]
	int    turn;
	__device__ __forceinline__ explicit row_sums(float* lds_) : lds(lds_), turn(0) {}
	__device__ __forceinline__ void operator()(float& x, float& y) {
		x = wave_sum(x), y = wave_sum(y);
		if constexpr(TPR > 64) {
			float* const at = lds + turn * (TPR / 64) * 2;
			turn ^= 1;
			if((threadIdx.x & 63) == 0) at[2 * (threadIdx.x >> 6)] = x, at[2 * (threadIdx.x >> 6) + 1] = y;
			__syncthreads();
			x = y = 0.f;
#pragma unroll
			for(int w = 0; w < TPR / 64; w++) x += at[2 * w], y += at[2 * w + 1];
		}
	}
	__device__ __forceinline__ float operator()(float x) {
		float none = 0.f;
		(*this)(x, none);
		return x;
	}
};

struct args {
	af3_residual_norm_params p;
	af3_residual_norm_grads  g;
	float   inv_c;
	int64_t per;       // backward: rows of a workgroup
	int64_t group;     // ... within (or a whole number of) stretches of this many rows
	uint32_t parts;    // ... workgroups per stretch, 0: stretches per workgroup instead
	float*  partial[4];   // a workgroup's sums [workgroups][C] for the gradients of gate, weight, bias, post_weight; null: none, or written where they belong
};

__device__ __forceinline__ int64_t share_row(int32_t share, int64_t row, int64_t group) { return share == AF3_SHARE_ROW ? row : share == AF3_SHARE_GROUP ? row / group : 0; }

// v -> (v - mean) / root and what that took, of a row held as floats
template <int NP, typename R, typename S>
__device__ __forceinline__ void standardise(float (&v)[NP][E], const R& row, S& sums, int32_t kind, float inv_c, float eps, float& mean, float& root) {
	mean = 0.f;
	if(kind == AF3_NORM_LAYER) {
		float s = 0.f;
#pragma unroll
		for(int n = 0; n < NP; n++)
#pragma unroll
			for(int e = 0; e < E; e++) s += v[n][e];
		mean = sums(s) * inv_c;
#pragma unroll
		for(int n = 0; n < NP; n++)
#pragma unroll
			for(int e = 0; e < E; e++) v[n][e] = row.in(n, e) ? v[n][e] - mean : 0.f;
	}
	float s = 0.f;
#pragma unroll
	for(int n = 0; n < NP; n++)
#pragma unroll
		for(int e = 0; e < E; e++) s = __builtin_fmaf(v[n][e], v[n][e], s);
	root = 1.f / __builtin_sqrtf(__builtin_fmaf(sums(s), inv_c, eps));
#pragma unroll
	for(int n = 0; n < NP; n++)
#pragma unroll
		for(int e = 0; e < E; e++) v[n][e] *= root;
}

constexpr int threads_for(int tpr) { return tpr == 64 ? 256 : tpr; }   // (wavefronts that have rows of their own need no barriers, others do)

template <typename T, int TPR, int NP>
__global__ void __launch_bounds__(threads_for(TPR)) forward_kernel(args a) {
	const af3_residual_norm_params& p = a.p;
	constexpr int AT_ONCE = threads_for(TPR) / TPR;
	__shared__ float lds[TPR > 64 ? 4 * (TPR / 64) : 1];
	const int64_t row = (blockIdx.y * (int64_t)gridDim.x + blockIdx.x) * AT_ONCE + threadIdx.x / TPR;
	if(row >= p.rows) return;   // (a whole wavefront, and with more of them to a row the whole workgroup)
	const row_of<T, TPR, NP> own(threadIdx.x % TPR, (int)p.C);
	row_sums<TPR>            sums(lds);
	const int64_t C = p.C;
	eight<T> y[NP], x[NP], m[NP];
	own.load(y, static_cast<const T*>(p.y) + row * p.y_stride);
	if(p.x) own.load(x, static_cast<const T*>(p.x) + row * p.x_stride);
	float r[NP][E];
#pragma unroll
	for(int n = 0; n < NP; n++)
#pragma unroll
		for(int e = 0; e < E; e++) r[n][e] = value(y[n].e[e]);
	f32x4 stats = {0.f, 0.f, 0.f, 0.f};
	if(p.post_norm != AF3_NORM_NONE) {
		float mean, root;
		standardise(r, own, sums, p.post_norm, a.inv_c, p.eps, mean, root);
		stats[0] = mean, stats[1] = root;
		if(p.post_weight) {
			own.load(m, static_cast<const T*>(p.post_weight));
#pragma unroll
			for(int n = 0; n < NP; n++)
#pragma unroll
				for(int e = 0; e < E; e++) r[n][e] *= value(m[n].e[e]);
		}
	}
	if(p.gate) {
		own.load(m, static_cast<const T*>(p.gate) + share_row(p.gate_share, row, p.group) * C);
#pragma unroll
		for(int n = 0; n < NP; n++)
#pragma unroll
			for(int e = 0; e < E; e++) r[n][e] *= p.gate_sigmoid ? sigmoidf_fast(value(m[n].e[e])) : value(m[n].e[e]);
	}
	if(p.x) {
#pragma unroll
		for(int n = 0; n < NP; n++)
#pragma unroll
			for(int e = 0; e < E; e++) r[n][e] = __builtin_fmaf(p.residual_scale, value(x[n].e[e]), r[n][e]);
	}
	own.store(static_cast<T*>(p.out) + row * C, r);
	if(p.norm != AF3_NORM_NONE) {
		float mean, root;
		standardise(r, own, sums, p.norm, a.inv_c, p.eps, mean, root);
		stats[2] = mean, stats[3] = root;
		if(p.weight) {
			own.load(m, static_cast<const T*>(p.weight) + share_row(p.weight_share, row, p.group) * C);
#pragma unroll
			for(int n = 0; n < NP; n++)
#pragma unroll
				for(int e = 0; e < E; e++) r[n][e] *= value(m[n].e[e]);
		}
		if(p.bias) {
			own.load(m, static_cast<const T*>(p.bias) + share_row(p.bias_share, row, p.group) * C);
#pragma unroll
			for(int n = 0; n < NP; n++)
#pragma unroll
				for(int e = 0; e < E; e++) r[n][e] += value(m[n].e[e]);
		}
		own.store(static_cast<T*>(p.normed) + row * C, r);
	}
	if(p.stats && threadIdx.x % TPR == 0) *reinterpret_cast<f32x4*>(p.stats + 4 * row) = stats;
}

// the gradient through v -> normed = (v - mean) root: g -> root (g - mean(g) - normed mean(g normed)), the mean of g for the layer norm alone
template <int NP, typename R, typename S>
__device__ __forceinline__ void back(float (&g)[NP][E], const float (&normed)[NP][E], const R& row, S& sums, int32_t kind, float inv_c, float root) {
	float s = 0.f, d = 0.f;
#pragma unroll
	for(int n = 0; n < NP; n++)
#pragma unroll
		for(int e = 0; e < E; e++) s += g[n][e], d = __builtin_fmaf(g[n][e], normed[n][e], d);
	sums(s, d);
	s = kind == AF3_NORM_LAYER ? s * inv_c : 0.f, d *= inv_c;
#pragma unroll
	for(int n = 0; n < NP; n++)
#pragma unroll
		for(int e = 0; e < E; e++) g[n][e] = row.in(n, e) ? root * (g[n][e] - s - normed[n][e] * d) : 0.f;
}

enum { GATE, WEIGHT, BIAS, POST };

// SUMS: some gradient is summed over rows
template <typename T, int TPR, int NP, bool SUMS>
__global__ void __launch_bounds__(threads_for(TPR)) backward_kernel(args a) {
	const af3_residual_norm_params& p = a.p;
	const af3_residual_norm_grads&  g = a.g;
	constexpr int AT_ONCE = threads_for(TPR) / TPR;
	__shared__ float lds[TPR > 64 ? 4 * (TPR / 64) : 1];
	__shared__ float joint[SUMS && AT_ONCE > 1 ? AT_ONCE * E * TPR * NP : 1];
	const int worker = threadIdx.x / TPR, lane = threadIdx.x % TPR;
	const row_of<T, TPR, NP> own(lane, (int)p.C);
	row_sums<TPR>            sums(lds);
	const int64_t C = p.C;

	int64_t first, last, step;   // rows of this workgroup; rows that share a group's row among them
	const int64_t block = blockIdx.y * (int64_t)gridDim.x + blockIdx.x;
	if(a.parts) {
		const int64_t stretch = block / a.parts, part = block - stretch * a.parts;
		first = stretch * a.group + part * a.per, last = first + a.per < (stretch + 1) * a.group ? first + a.per : (stretch + 1) * a.group;
		step  = a.per;
	} else {
		first = block * a.per, last = first + a.per < p.rows ? first + a.per : p.rows;
		step  = a.group;
	}
	if(first >= p.rows) return;   // (the whole workgroup)
	float total[SUMS ? 4 : 1][NP][E];
	auto  clear = [&](int which) {
#pragma unroll
		for(int n = 0; n < NP; n++)
#pragma unroll
			for(int e = 0; e < E; e++) total[which][n][e] = 0.f;
	};
	// a finished sum: the workgroup's part of it, or, where the workgroup has all of it, the gradient's row
	auto flush = [&](int which, float* part, T* result) {
		if constexpr(AT_ONCE > 1) {
			__syncthreads();
			own.store_sums(joint + worker * (E * TPR * NP), total[which]);
			__syncthreads();
			if(worker == 0) {
#pragma unroll
				for(int n = 0; n < NP; n++)
#pragma unroll
					for(int e = 0; e < E; e++)
						if(own.in(n, e)) {
							float s = 0.f;
#pragma unroll
							for(int w = 0; w < AT_ONCE; w++) s += joint[w * (E * TPR * NP) + own.at(n) + e];
							total[which][n][e] = s;
						}
			}
		}
		if(worker == 0) {
			if(part) own.store_sums(part, total[which]);
			else own.store(result, total[which]);
		}
	};
	if constexpr(SUMS) clear(GATE), clear(WEIGHT), clear(BIAS), clear(POST);

	// What a row needs comes in one go, a row ahead of its use where the registers hold two of them; what rows share stays in registers.  4 x 2048 rows of 4096 channels in bf16:
	// 107 us (six tensors of 67 MB and 25 of workgroups' sums: 4.0 TB/s); with 16 channels a thread, everything loaded where it is used, 210; 8 x 768 conditioned rows of 768 channels 29 us
	// (104 MB: 3.6 TB/s), that way 54.  Vector instructions take 67 % of the SIMDs' clocks and wavefronts wait 39 % of theirs: two to a SIMD, one row at a time, a barrier for each norm's sums.
	constexpr bool AHEAD = TPR * NP <= 1024;
	struct streams {
		eight<T> y[NP], x[NP], out[NP], normed[NP], gate[NP], weight[NP];
		f32x4    stats;
	} coming;
	const bool through = p.norm != AF3_NORM_NONE && g.grad_normed;   // a gradient comes through the second norm
	eight<T> post[NP];
	if(p.post_weight) own.load(post, static_cast<const T*>(p.post_weight));
	auto shared = [&](int64_t row) {
		if(p.gate && p.gate_share != AF3_SHARE_ROW) own.load(coming.gate, static_cast<const T*>(p.gate) + share_row(p.gate_share, row, p.group) * C);
		if(p.weight && p.weight_share != AF3_SHARE_ROW) own.load(coming.weight, static_cast<const T*>(p.weight) + share_row(p.weight_share, row, p.group) * C);
	};
	auto fetch = [&](int64_t row) {
		own.load(coming.y, static_cast<const T*>(p.y) + row * p.y_stride);
		if(through) {
			if(p.x) own.load(coming.x, static_cast<const T*>(p.x) + row * p.x_stride);
			own.load(coming.normed, static_cast<const T*>(g.grad_normed) + row * g.grad_normed_stride);
			if(p.weight_share == AF3_SHARE_ROW) own.load(coming.weight, static_cast<const T*>(p.weight) + row * C);
		}
		if(g.grad_out) own.load(coming.out, static_cast<const T*>(g.grad_out) + row * g.grad_out_stride);
		if(p.gate_share == AF3_SHARE_ROW) own.load(coming.gate, static_cast<const T*>(p.gate) + row * C);
		coming.stats = *reinterpret_cast<const f32x4*>(p.stats + 4 * row);
	};
	for(int64_t begin = first; begin < last; begin += step) {
		const int64_t end = begin + step < last ? begin + step : last;
		if(begin + worker < end) {
			shared(begin);
			if(AHEAD) fetch(begin + worker);
		}
		for(int64_t row = begin + worker; row < end; row += AT_ONCE) {
			if(!AHEAD) fetch(row);
			const streams s = coming;
			if(AHEAD && row + AT_ONCE < end) fetch(row + AT_ONCE);
			const f32x4 stats = s.stats;
			float       z[NP][E], gate[NP][E], r[NP][E], d[NP][E];   // d: the gradient on its way back
			// the forward pass again: z = normed y, r = its sum, standardised
#pragma unroll
			for(int n = 0; n < NP; n++)
#pragma unroll
				for(int e = 0; e < E; e++) {
					z[n][e] = value(s.y[n].e[e]), d[n][e] = 0.f;
					if(p.post_norm != AF3_NORM_NONE) z[n][e] = own.in(n, e) ? (z[n][e] - stats[0]) * stats[1] : 0.f;
					gate[n][e] = !p.gate ? 1.f : p.gate_sigmoid ? sigmoidf_fast(value(s.gate[n].e[e])) : value(s.gate[n].e[e]);
				}
			auto after = [&](int n, int e) { return p.post_weight ? z[n][e] * value(post[n].e[e]) : z[n][e]; };   // what the gate is multiplied with
			if(through) {
#pragma unroll
				for(int n = 0; n < NP; n++)
#pragma unroll
					for(int e = 0; e < E; e++) {
						r[n][e] = gate[n][e] * after(n, e);
						if(p.x) r[n][e] = __builtin_fmaf(p.residual_scale, value(s.x[n].e[e]), r[n][e]);
						r[n][e] = own.in(n, e) ? (r[n][e] - stats[2]) * stats[3] : 0.f;
						d[n][e] = value(s.normed[n].e[e]);
					}
				if(g.grad_bias) {
					if(p.bias_share == AF3_SHARE_ROW) own.store(static_cast<T*>(g.grad_bias) + row * C, d);
					else if constexpr(SUMS) {
#pragma unroll
						for(int n = 0; n < NP; n++)
#pragma unroll
							for(int e = 0; e < E; e++) total[BIAS][n][e] += d[n][e];
					}
				}
				if(g.grad_weight) {
					if(p.weight_share == AF3_SHARE_ROW) {
						float w[NP][E];
#pragma unroll
						for(int n = 0; n < NP; n++)
#pragma unroll
							for(int e = 0; e < E; e++) w[n][e] = d[n][e] * r[n][e];
						own.store(static_cast<T*>(g.grad_weight) + row * C, w);
					} else if constexpr(SUMS) {
#pragma unroll
						for(int n = 0; n < NP; n++)
#pragma unroll
							for(int e = 0; e < E; e++) total[WEIGHT][n][e] = __builtin_fmaf(d[n][e], r[n][e], total[WEIGHT][n][e]);
					}
				}
				if(p.weight) {
#pragma unroll
					for(int n = 0; n < NP; n++)
#pragma unroll
						for(int e = 0; e < E; e++) d[n][e] *= value(s.weight[n].e[e]);
				}
				back(d, r, own, sums, p.norm, a.inv_c, stats[3]);
			}
			if(g.grad_out) {
#pragma unroll
				for(int n = 0; n < NP; n++)
#pragma unroll
					for(int e = 0; e < E; e++) d[n][e] += value(s.out[n].e[e]);
			}
			if(g.grad_x) {
				float dx[NP][E];
#pragma unroll
				for(int n = 0; n < NP; n++)
#pragma unroll
					for(int e = 0; e < E; e++) dx[n][e] = p.residual_scale * d[n][e];
				own.store(static_cast<T*>(g.grad_x) + row * C, dx);
			}
			if(g.grad_gate) {
				float dg[NP][E];
#pragma unroll
				for(int n = 0; n < NP; n++)
#pragma unroll
					for(int e = 0; e < E; e++) dg[n][e] = d[n][e] * after(n, e) * (p.gate_sigmoid ? gate[n][e] * (1.f - gate[n][e]) : 1.f);
				if(p.gate_share == AF3_SHARE_ROW) own.store(static_cast<T*>(g.grad_gate) + row * C, dg);
				else if constexpr(SUMS) {
#pragma unroll
					for(int n = 0; n < NP; n++)
#pragma unroll
						for(int e = 0; e < E; e++) total[GATE][n][e] += dg[n][e];
				}
			}
#pragma unroll
			for(int n = 0; n < NP; n++)
#pragma unroll
				for(int e = 0; e < E; e++) d[n][e] *= gate[n][e];
			if constexpr(SUMS)
				if(g.grad_post_weight) {
#pragma unroll
					for(int n = 0; n < NP; n++)
#pragma unroll
						for(int e = 0; e < E; e++) total[POST][n][e] = __builtin_fmaf(d[n][e], z[n][e], total[POST][n][e]);
				}
			if(g.grad_y) {
				if(p.post_norm != AF3_NORM_NONE) {
					if(p.post_weight) {
#pragma unroll
						for(int n = 0; n < NP; n++)
#pragma unroll
							for(int e = 0; e < E; e++) d[n][e] *= value(post[n].e[e]);
					}
					back(d, z, own, sums, p.post_norm, a.inv_c, stats[1]);
				}
				own.store(static_cast<T*>(g.grad_y) + row * C, d);
			}
		}
		if constexpr(SUMS) {   // what the rows of a group share
			auto group_sum = [&](int which, int32_t share, void* result) {
				if(!result || share != AF3_SHARE_GROUP) return;
				flush(which, a.partial[which] ? a.partial[which] + block * C : nullptr, static_cast<T*>(result) + begin / p.group * C);
				clear(which);
			};
			group_sum(GATE, p.gate_share, g.grad_gate), group_sum(WEIGHT, p.weight_share, g.grad_weight), group_sum(BIAS, p.bias_share, g.grad_bias);
		}
	}
	if constexpr(SUMS) {
		auto sum = [&](int which, int32_t share, void* result) {
			if(result && share == AF3_SHARE_CHANNEL) flush(which, a.partial[which] + block * C, nullptr);
		};
		sum(GATE, p.gate_share, g.grad_gate), sum(WEIGHT, p.weight_share, g.grad_weight), sum(BIAS, p.bias_share, g.grad_bias), sum(POST, AF3_SHARE_CHANNEL, g.grad_post_weight);
	}
}

// The workgroups' sums joined: result row i of `n[which]` is the sum of `parts` consecutive rows of the partial sums.  A workgroup has 64 channels, 4 to a thread; its 16
// rows of threads take the parts in turn.
struct join_args {
	const float* partial[4];
	void*        out[4];
	uint32_t     parts[4], rows[4];
	uint32_t     columns;   // workgroups per row
	int32_t      C, dtype;
};
__global__ void __launch_bounds__(256) join_kernel(join_args a) {
	__shared__ f32x4 joint[16][16];
	uint32_t block = blockIdx.x;
	int      which = 0;
	while(which < 3 && block >= a.rows[which] * a.columns) block -= a.rows[which++] * a.columns;
	const uint32_t row = block / a.columns, lane = threadIdx.x & 15, turn = threadIdx.x >> 4;
	const int      c = 64 * (int)(block - row * a.columns) + 4 * (int)lane;
	const float*   at = a.partial[which] + (int64_t)row * a.parts[which] * a.C + c;
	f32x4          sum = {0.f, 0.f, 0.f, 0.f};
	const uint32_t parts = a.parts[which];
	if(c + 4 <= a.C) {
#pragma unroll 8
		for(uint32_t i = turn; i < parts; i += 16) sum += *reinterpret_cast<const f32x4_any*>(at + (int64_t)i * a.C);
	} else {
		for(uint32_t i = turn; i < parts; i += 16)
			for(int e = 0; e < 4; e++)
				if(c + e < a.C) sum[e] += at[(int64_t)i * a.C + e];
	}
	joint[turn][lane] = sum;
	__syncthreads();
	if(turn != 0) return;
#pragma unroll
	for(int i = 1; i < 16; i++) sum += joint[i][lane];
	for(int e = 0; e < 4; e++) {
		if(c + e >= a.C) break;
		const int64_t to = (int64_t)row * a.C + c + e;
		if(a.dtype == AF3_F32) static_cast<float*>(a.out[which])[to] = sum[e];
		else static_cast<uint16_t*>(a.out[which])[to] = bits<uint16_t>(sum[e]);
	}
}

// ---- host side -------------------------------------------------------------------------------------------------------------
// f(threads per row, stretches of 8 channels per thread).  Forward: as few wavefronts to a row as hold it in 16 channels a thread, a workgroup where the rows are few; backward,
// which holds three times as much of a row and the sums: 8 channels a thread as far as workgroups go.
template <typename F>
int with_shape(int64_t C, int64_t rows, F f) {
	if(C <= 512) return f(ic<64>(), ic<1>());
	if(C <= 1024 && rows >= 2048) return f(ic<64>(), ic<2>());
	if(C <= 2048) return f(ic<256>(), ic<1>());
	if(C <= 4096) return f(ic<256>(), ic<2>());
	if(C <= 8192) return f(ic<512>(), ic<2>());
	return f(ic<1024>(), ic<2>());
}
template <typename F>
int with_backward_shape(int64_t C, F f) {
	if(C <= 512) return f(ic<64>(), ic<1>());
	if(C <= 1024) return f(ic<128>(), ic<1>());
	if(C <= 2048) return f(ic<256>(), ic<1>());
	if(C <= 4096) return f(ic<512>(), ic<1>());
	if(C <= 8192) return f(ic<1024>(), ic<1>());
	return f(ic<1024>(), ic<2>());
}
inline int64_t over(int64_t n, int64_t per) { return (n + per - 1) / per; }

template <typename T>
int forward(const args& a, hipStream_t s) {
	return with_shape(a.p.C, a.p.rows, [&](auto tpr, auto np) {
		constexpr int TPR = decltype(tpr)::value, NP = decltype(np)::value, THREADS = threads_for(TPR);
		hipLaunchKernelGGL((forward_kernel<T, TPR, NP>), grid_of(over(a.p.rows, THREADS / TPR)), dim3(THREADS), 0, s, a);
		return launch_status();
	});
}

// how the rows are dealt out, and which sums go by way of the workspace
struct plan {
	int64_t  per, group;
	uint32_t parts, workgroups;
	bool     sums;
	bool     partial[4];
	uint32_t joined[4], rows[4];   // partial sums per result row, result rows
	int64_t  floats;               // of the workspace
};
plan backward_plan(const af3_residual_norm_params& p, const af3_residual_norm_grads& g) {
	plan f{};
	const int32_t share[4] = {p.gate_share, p.weight_share, p.bias_share, AF3_SHARE_CHANNEL};
	const void*   wanted[4] = {g.grad_gate, g.grad_weight, g.grad_bias, g.grad_post_weight};
	bool          grouped = p.gate_share == AF3_SHARE_GROUP || p.weight_share == AF3_SHARE_GROUP;   // (rows that are read once for a group, whether their gradient is wanted or not)
	for(int i = 0; i < 4; i++)
		if(wanted[i] && share[i] != AF3_SHARE_ROW) f.sums = true, grouped = grouped || share[i] == AF3_SHARE_GROUP;
	f.group = grouped ? p.group : p.rows;
	// With sums: about as many workgroups as fit the chip together, so that their parts' way through memory stays small beside the rows'; without: a few rows to a worker.
	const int64_t at_once = p.C <= 512 ? 4 : 1, most = p.C <= 512 ? 1024 : p.C <= 1024 ? 2048 : p.C <= 2048 ? 1024 : p.C <= 4096 ? 512 : 256;
	const int64_t target = f.sums ? over(over(p.rows, most), at_once) * at_once : 4 * at_once;
	if(f.group >= target) {
		f.parts = (uint32_t)over(f.group, target), f.per = over(f.group, f.parts);
		f.workgroups = (uint32_t)(p.rows / f.group) * f.parts;
	} else {
		f.parts = 0, f.per = target / f.group * f.group;
		f.workgroups = (uint32_t)over(p.rows, f.per);
	}
	for(int i = 0; i < 4; i++) {
		if(!wanted[i] || share[i] == AF3_SHARE_ROW) continue;
		if(share[i] == AF3_SHARE_GROUP) {
			if(f.parts <= 1) continue;   // (a workgroup has all of a group's rows)
			f.joined[i] = f.parts, f.rows[i] = (uint32_t)(p.rows / p.group);
		} else {
			f.joined[i] = f.workgroups, f.rows[i] = 1;
		}
		f.partial[i] = true, f.floats += over((int64_t)f.workgroups * p.C, 4) * 4;
	}
	return f;
}

template <typename T>
int backward(const args& a, const plan& f, hipStream_t s) {
	return with_backward_shape(a.p.C, [&](auto tpr, auto np) {
		constexpr int TPR = decltype(tpr)::value, NP = decltype(np)::value, THREADS = threads_for(TPR);
		if(f.sums) hipLaunchKernelGGL((backward_kernel<T, TPR, NP, true>), grid_of(f.workgroups), dim3(THREADS), 0, s, a);
		else hipLaunchKernelGGL((backward_kernel<T, TPR, NP, false>), grid_of(f.workgroups), dim3(THREADS), 0, s, a);
		return launch_status();
	});
}

int validate(const af3_residual_norm_params* p) {
	if(!p) return AF3_ERR_NULL_POINTER;
	if(p->dtype != AF3_F32 && p->dtype != AF3_BF16) return AF3_ERR_BAD_DTYPE;
	if(p->rows <= 0 || p->rows > 0x3fffffff || p->C <= 0 || p->C > AF3_RESIDUAL_NORM_MAX_CHANNELS) return AF3_ERR_BAD_SHAPE;
	if(!p->y) return AF3_ERR_NULL_POINTER;
	if(p->norm < AF3_NORM_NONE || p->norm > AF3_NORM_LAYER || p->post_norm < AF3_NORM_NONE || p->post_norm > AF3_NORM_LAYER) return AF3_ERR_BAD_ARGUMENT;
	if(p->norm == AF3_NORM_NONE && (p->weight || p->bias)) return AF3_ERR_BAD_ARGUMENT;
	if(p->post_norm == AF3_NORM_NONE && p->post_weight) return AF3_ERR_BAD_ARGUMENT;
	const void*   of[3] = {p->gate, p->weight, p->bias};
	const int32_t share[3] = {p->gate_share, p->weight_share, p->bias_share};
	for(int i = 0; i < 3; i++) {
		if(share[i] < AF3_SHARE_NONE || share[i] > AF3_SHARE_ROW || (share[i] == AF3_SHARE_NONE) != (of[i] == nullptr)) return AF3_ERR_BAD_ARGUMENT;
		if(share[i] == AF3_SHARE_GROUP && (p->group <= 0 || p->rows % p->group != 0)) return AF3_ERR_BAD_SHAPE;
	}
	if(p->y_stride < 0 || (p->x && p->x_stride < 0)) return AF3_ERR_BAD_STRIDE;
	if(!(p->eps >= 0.f) || !(p->eps < INFINITY) || !(p->residual_scale - p->residual_scale == 0.f)) return AF3_ERR_BAD_ARGUMENT;
	return AF3_OK;
}
int validate_grads(const af3_residual_norm_params* p, const af3_residual_norm_grads* g) {
	if(const int rc = validate(p); rc != AF3_OK) return rc;
	if(!g || (!g->grad_out && !g->grad_normed)) return AF3_ERR_NULL_POINTER;
	if((g->grad_x && !p->x) || (g->grad_gate && !p->gate) || (g->grad_weight && !p->weight) || (g->grad_bias && !p->bias) || (g->grad_post_weight && !p->post_weight)) return AF3_ERR_NULL_POINTER;
	if((g->grad_weight || g->grad_bias) && !g->grad_normed) return AF3_ERR_NULL_POINTER;   // (zeros, which the caller writes)
	if(g->grad_normed && p->norm == AF3_NORM_NONE) return AF3_ERR_BAD_ARGUMENT;
	if(!g->grad_x && !g->grad_y && !g->grad_gate && !g->grad_weight && !g->grad_bias && !g->grad_post_weight) return AF3_ERR_NULL_POINTER;
	if(g->grad_out_stride < 0 || g->grad_normed_stride < 0) return AF3_ERR_BAD_STRIDE;
	return AF3_OK;
}

}  // namespace rnorm
}  // namespace af3

using namespace af3;

extern "C" int af3_residual_norm_forward(const af3_residual_norm_params* params, void* hip_stream) {
	if(const int rc = rnorm::validate(params); rc != AF3_OK) return rc;
	if(!params->out || (params->norm != AF3_NORM_NONE) != (params->normed != nullptr)) return AF3_ERR_NULL_POINTER;
	if(reinterpret_cast<uintptr_t>(params->stats) & 15) return AF3_ERR_BAD_ARGUMENT;
	if(const int dc = current_device_status(); dc != AF3_OK) return dc;
	rnorm::args a{};
	a.p = *params, a.inv_c = 1.f / (float)params->C;
	const hipStream_t s = static_cast<hipStream_t>(hip_stream);
	return params->dtype == AF3_F32 ? rnorm::forward<float>(a, s) : rnorm::forward<uint16_t>(a, s);
}

extern "C" int64_t af3_residual_norm_backward_workspace_bytes(const af3_residual_norm_params* params, const af3_residual_norm_grads* grads) {
	const int rc = rnorm::validate_grads(params, grads);
	return rc != AF3_OK ? rc : rnorm::backward_plan(*params, *grads).floats * 4;
}

extern "C" int af3_residual_norm_backward(const af3_residual_norm_params* params, const af3_residual_norm_grads* grads, void* hip_stream) {
	if(const int rc = rnorm::validate_grads(params, grads); rc != AF3_OK) return rc;
	if(!params->stats) return AF3_ERR_NULL_POINTER;
	if(reinterpret_cast<uintptr_t>(params->stats) & 15) return AF3_ERR_BAD_ARGUMENT;
	const rnorm::plan f = rnorm::backward_plan(*params, *grads);
	if(f.floats > 0 && (!grads->workspace || grads->workspace_bytes < f.floats * 4 || (reinterpret_cast<uintptr_t>(grads->workspace) & 15))) return AF3_ERR_BAD_ARGUMENT;
	if(const int dc = current_device_status(); dc != AF3_OK) return dc;
	rnorm::args a{};
	a.p = *params, a.g = *grads, a.inv_c = 1.f / (float)params->C, a.per = f.per, a.group = f.group, a.parts = f.parts;
	rnorm::join_args j{};
	void* const results[4] = {grads->grad_gate, grads->grad_weight, grads->grad_bias, grads->grad_post_weight};
	float*      space = static_cast<float*>(grads->workspace);
	uint32_t    joins = 0;
	j.columns = (uint32_t)rnorm::over(params->C, 64), j.C = (int32_t)params->C, j.dtype = params->dtype;
	for(int i = 0; i < 4; i++) {
		if(!f.partial[i]) continue;
		a.partial[i] = space, space += rnorm::over((int64_t)f.workgroups * params->C, 4) * 4;
		j.partial[i] = a.partial[i], j.out[i] = results[i], j.parts[i] = f.joined[i], j.rows[i] = f.rows[i];
		joins += f.rows[i] * j.columns;
	}
	const hipStream_t s = static_cast<hipStream_t>(hip_stream);
	const int rc = params->dtype == AF3_F32 ? rnorm::backward<float>(a, f, s) : rnorm::backward<uint16_t>(a, f, s);
	if(rc != AF3_OK || joins == 0) return rc;
	hipLaunchKernelGGL(rnorm::join_kernel, dim3(joins), dim3(256), 0, s, j);
	return launch_status();
}
