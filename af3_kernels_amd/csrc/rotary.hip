// Rotary positions: pair i of a head's first `rotary` elements is turned by the angle a = position * frequency[i],
//     (x, y) -> scale (x cos a - y sin a, x sin a + y cos a),
// the rest of the head goes through as it is.  Pairs are elements (i, i + rotary / 2), or (2 i, 2 i + 1) where interleaved.  The gradient is the same with -a.
// af3_rotary_embedding.
//
// Reads and writes the heads once and nothing else to speak of: cosines and sines are worked out where they are used.  A thread has the same few pairs of one token for
// several heads, so that an angle's ~50 instructions (64 bits up to the part of a turn: at position 10^6 a float would leave 2^-4 of it) serve them all.
// 4 x (32 + 8) x 4096 x 128 in bf16: 67.7 us, 4.96 TB/s, what a large copy reaches; one token of 32 requests 5.4 us, which is a launch.
#include "mfma_helpers.hpp"

namespace af3 {
namespace rotary {

constexpr int THREADS = 256;

struct args {
	af3_rotary_params p;
	uint32_t turned, units;   // units of 2 V elements of a head: those that are turned, all of them
	uint32_t tokens, per;     // B * L; heads per thread
};

template <int BYTES>
struct raw;
template <> struct raw<32> { typedef struct { u32x4_any a, b; } type; };
template <> struct raw<16> { typedef u32x4_any type; };
template <> struct raw<8> { typedef u32x2_any type; };
template <> struct raw<4> { typedef __attribute__((aligned(2))) uint32_t type; };
template <> struct raw<2> { typedef uint16_t type; };

template <typename T> __device__ __forceinline__ float value(T x);
template <> __device__ __forceinline__ float value<uint16_t>(uint16_t x) { return bf16_bits_to_f32(x); }
template <> __device__ __forceinline__ float value<float>(float x) { return x; }
template <typename T> __device__ __forceinline__ T bits(float x);
template <> __device__ __forceinline__ uint16_t bits<uint16_t>(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
template <> __device__ __forceinline__ float bits<float>(float x) { return x; }

// V elements side by side, at any element's address
template <typename T, int V>
struct piece {
	T e[V];
	__device__ __forceinline__ void load(const T* p) {
		const auto v = *reinterpret_cast<const typename raw<V * sizeof(T)>::type*>(p);
		__builtin_memcpy(e, &v, sizeof(e));
	}
	__device__ __forceinline__ void store(T* p) const {
		typename raw<V * sizeof(T)>::type v;
		__builtin_memcpy(&v, e, sizeof(e));
		*reinterpret_cast<typename raw<V * sizeof(T)>::type*>(p) = v;
	}
};

template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS) rotary_kernel(args a) {
	const af3_rotary_params& p = a.p;
	constexpr int  AT_ONCE = 4;   // heads whose loads are in flight together
	const uint32_t at = blockIdx.x * THREADS + threadIdx.x;
	const uint32_t token = at / a.units, u = at - token * a.units;
	if(token >= a.tokens) return;
	const uint32_t b = token / (uint32_t)p.L, l = token - b * (uint32_t)p.L;
	const int      heads = (int)(p.heads[0] + p.heads[1]), D = (int)p.D, n = (int)p.rotary;
	const int      first = (int)(blockIdx.y * a.per), last = first + (int)a.per < heads ? first + (int)a.per : heads;
	const bool     turns = u < a.turned;
	// where the unit's two pieces begin
	const int d0 = turns ? (INTERLEAVED ? 2 * V * (int)u : V * (int)u) : n + 2 * V * (int)(u - a.turned), d1 = turns && !INTERLEAVED ? d0 + n / 2 : d0 + V;

	auto row = [&](int h, bool out) -> T* {
		const int     of = h < p.heads[0] ? 0 : 1, i = of ? h - (int)p.heads[0] : h;
		const int64_t* st = out ? p.out_stride[of] : p.x_stride[of];
		return static_cast<T*>(out ? p.out[of] : const_cast<void*>(p.x[of])) + b * st[0] + i * st[1] + l * st[2];
	};
	if(!turns && d0 + 2 * V > D) {   // the end of a head whose untouched part is no whole number of units
		for(int h = first; h < last; h++)
			for(int d = d0; d < D; d++) row(h, true)[d] = row(h, false)[d];
		return;
	}
	piece<T, V> x[AT_ONCE], y[AT_ONCE];
	auto fetch = [&](int h0) {
#pragma unroll
		for(int i = 0; i < AT_ONCE; i++)
			if(h0 + i < last) x[i].load(row(h0 + i, false) + d0), y[i].load(row(h0 + i, false) + d1);
	};
	fetch(first);   // (on their way while the angles are worked out)
	float c[V], s[V];
	if(turns) {
		const int64_t position = p.positions ? p.positions[b * p.position_stride_b + l] : p.offset + (int64_t)l;
		const double  turn = (double)position * 0.15915494309189533576888;
#pragma unroll
		for(int i = 0; i < V; i++) {
			const double t = turn * p.frequencies[V * u + i];
			sincospif(2.f * (float)(t - __builtin_rint(t)), &s[i], &c[i]);
			c[i] *= p.scale, s[i] *= p.inverse ? -p.scale : p.scale;
		}
	}
	for(int h0 = first; h0 < last; h0 += AT_ONCE) {
		piece<T, V> to_x[AT_ONCE], to_y[AT_ONCE];
#pragma unroll
		for(int i = 0; i < AT_ONCE; i++) {
			to_x[i] = x[i], to_y[i] = y[i];
			if(turns) {
#pragma unroll
				for(int e = 0; e < V; e++) {
					// (interleaved: pair e lies in elements 2 e, 2 e + 1 of the two pieces)
					const bool  second = INTERLEAVED && 2 * e >= V;
					const int   ea = INTERLEAVED ? (2 * e) % V : e, eb = INTERLEAVED ? (V == 1 ? 0 : (2 * e) % V + 1) : e;
					const bool  split = !INTERLEAVED || V == 1;   // (its halves are in one piece each)
					const float va = value<T>(split ? x[i].e[ea] : second ? y[i].e[ea] : x[i].e[ea]), vb = value<T>(split ? y[i].e[eb] : second ? y[i].e[eb] : x[i].e[eb]);
					const T     ra = bits<T>(__builtin_fmaf(va, c[e], -(vb * s[e]))), rb = bits<T>(__builtin_fmaf(va, s[e], vb * c[e]));
					if(split) to_x[i].e[ea] = ra, to_y[i].e[eb] = rb;
					else if(second) to_y[i].e[ea] = ra, to_y[i].e[eb] = rb;
					else to_x[i].e[ea] = ra, to_x[i].e[eb] = rb;
				}
			}
		}
		if(h0 + AT_ONCE < last) fetch(h0 + AT_ONCE);
#pragma unroll
		for(int i = 0; i < AT_ONCE; i++)
			if(h0 + i < last) to_x[i].store(row(h0 + i, true) + d0), to_y[i].store(row(h0 + i, true) + d1);
	}
}

template <typename T, int V>
int launch(args a, hipStream_t s) {
	const af3_rotary_params& p = a.p;
	const int64_t heads = p.heads[0] + p.heads[1];
	a.turned = (uint32_t)(p.rotary / (2 * V));
	a.units  = a.turned + (uint32_t)((p.D - p.rotary + 2 * V - 1) / (2 * V));
	const int64_t threads = (int64_t)a.tokens * a.units;
	// Few tokens: fewer heads per thread, so that the launch fills the chip (2^17 threads are two wavefronts to a SIMD).
	int64_t groups = threads >= (1 << 17) ? 1 : ((1 << 17) + threads - 1) / threads;
	if(groups > heads) groups = heads;
	a.per = (uint32_t)((heads + groups - 1) / groups);
	groups = (heads + a.per - 1) / a.per;
	const int64_t blocks = (threads + THREADS - 1) / THREADS;
	if(blocks > 0xffffff || groups > 0xffff) return AF3_ERR_BAD_SHAPE;
	const dim3 grid((uint32_t)blocks, (uint32_t)groups);
	if(p.interleaved) hipLaunchKernelGGL((rotary_kernel<T, V, true>), grid, dim3(THREADS), 0, s, a);
	else hipLaunchKernelGGL((rotary_kernel<T, V, false>), grid, dim3(THREADS), 0, s, a);
	return launch_status();
}
// as many pairs per thread as make 16-byte pieces, fewer where the pairs are no whole number of those
template <typename T>
int launch_type(const args& a, hipStream_t s) {
	const int64_t pairs = a.p.rotary / 2;
	if constexpr(sizeof(T) == 2)
		if(pairs % 8 == 0) return launch<T, 8>(a, s);
	if(pairs % 4 == 0) return launch<T, 4>(a, s);
	if(pairs % 2 == 0) return launch<T, 2>(a, s);
	return launch<T, 1>(a, s);
}

int validate(const af3_rotary_params* p) {
	if(!p || !p->x[0] || !p->out[0] || !p->frequencies) return AF3_ERR_NULL_POINTER;
	if(p->dtype != AF3_F32 && p->dtype != AF3_BF16) return AF3_ERR_BAD_DTYPE;
	if(p->B <= 0 || p->L <= 0 || p->D <= 0 || p->heads[0] <= 0 || p->heads[1] < 0) return AF3_ERR_BAD_SHAPE;
	if(p->D > AF3_ROTARY_MAX_HEAD_DIM || p->rotary <= 0 || p->rotary > p->D || p->rotary % 2 != 0) return AF3_ERR_BAD_SHAPE;
	if(p->heads[0] > 0xffff || p->heads[1] > 0xffff - p->heads[0] || p->B > 0x3fffffff || p->L > 0x3fffffff || p->B * p->L > 0x3fffffff) return AF3_ERR_BAD_SHAPE;
	if(p->heads[1] > 0 && (!p->x[1] || !p->out[1])) return AF3_ERR_NULL_POINTER;
	for(int i = 0; i < 2; i++) {
		if(p->heads[i] == 0) continue;
		for(int j = 0; j < 3; j++)
			if(p->x_stride[i][j] < 0 || p->out_stride[i][j] < 0) return AF3_ERR_BAD_STRIDE;
		// (inputs may repeat rows, results may not)
		if((p->L > 1 && p->out_stride[i][2] < p->D) || (p->heads[i] > 1 && p->out_stride[i][1] < p->D) || (p->B > 1 && p->out_stride[i][0] < p->D)) return AF3_ERR_BAD_STRIDE;
	}
	if(p->positions && p->position_stride_b < 0) return AF3_ERR_BAD_STRIDE;
	if(p->offset > ((int64_t)1 << 62) || p->offset < -((int64_t)1 << 62) || !(p->scale - p->scale == 0.f)) return AF3_ERR_BAD_ARGUMENT;
	return AF3_OK;
}

}  // namespace rotary
}  // namespace af3

extern "C" int af3_rotary_embedding(const af3_rotary_params* params, void* hip_stream) {
	using namespace af3;
	if(const int rc = rotary::validate(params); rc != AF3_OK) return rc;
	if(const int dc = current_device_status(); dc != AF3_OK) return dc;
	rotary::args a{};
	a.p = *params, a.tokens = (uint32_t)(params->B * params->L);
	const hipStream_t s = static_cast<hipStream_t>(hip_stream);
	return params->dtype == AF3_F32 ? rotary::launch_type<float>(a, s) : rotary::launch_type<uint16_t>(a, s);
}
