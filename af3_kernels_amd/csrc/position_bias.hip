// The learned relative position bias: out[h][q][k] = table[bucket(k_pos[k] - q_pos[q])][h], and the table's gradient, the sums of
// out's gradient by bucket.  af3_position_bias_forward, af3_position_bias_backward.
//
// A bucket is found by its smallest distance: `border` holds those of one side in ascending order, worked out on the host in whole
// numbers, so that no logarithm's rounding decides at a border.  From the last border on (`reach`) nothing changes any more: the
// buckets (backward) or the head's values (forward) of the offsets -reach .. reach are a table in LDS, and 16 bytes of keys that all
// lie beyond it are one value.  Both kernels are bound by memory: the forward pass writes, the backward pass reads H Lq Lk values.
#include "cross_tiles.hpp"

#include <math.h>

namespace af3 {
namespace position {

using cross::kind;
using cross::load16;
using cross::store16;

constexpr int MAX_BUCKETS = AF3_POSITION_BIAS_MAX_BUCKETS;
constexpr int MAX_OFFSETS = 4097;   // of the table in LDS; with more, buckets are searched for one by one
constexpr int THREADS = 256;

struct args {
	const void*    table;    // forward: the values; backward: not read
	void*          out;      // forward: [H, Lq, Lk]; backward: the table's gradient
	const void *   grad, *rest;   // backward: [H, Lq, Lk]; what its rounding lost, or null
	float*         partial;  // backward: [H][parts][buckets], with rest those of rest behind them
	const int64_t *q_pos, *k_pos;
	int64_t        q_offset;
	int64_t        table_stride[2], grad_stride[2];
	int64_t        H, Lq, Lk;
	int32_t        buckets, borders, reach;
	int32_t        first_behind, step_behind, first_ahead, step_ahead;   // bucket = first + step * (borders passed), keys behind (and at) the query and ahead of it
	int32_t        columns_log2, rows;   // threads across the columns of a workgroup, rows of a workgroup
	int32_t        near;                 // the first `near` borders are 1, 2, 3, ...
	int32_t        far_border[MAX_BUCKETS / 2];   // the others (arguments lie in host memory, and every workgroup reads what it needs of them from there)
};
// border i of a call
__device__ __forceinline__ int border_of(const args& a, int i) { return i < a.near ? i + 1 : a.far_border[i - a.near]; }

__device__ __forceinline__ int passed(const int* border, int n, int d) {   // how many borders are <= d
	int low = 0;
	while(n > 0) {
		const int half = n >> 1;
		if(border[low + half] <= d) low += half + 1, n -= half + 1;
		else n = half;
	}
	return low;
}
__device__ __forceinline__ int bucket_of(const args& a, const int* border, int rel) {
	return rel <= 0 ? a.first_behind + a.step_behind * passed(border, a.borders, -rel) : a.first_ahead + a.step_ahead * passed(border, a.borders, rel);
}
// put(offset, bucket) for all offsets -reach .. reach: thread t writes those between border t - 1 and border t
template <int N, typename F>
__device__ __forceinline__ void for_all_offsets(const args& a, const int* border, F put) {
	for(int t = threadIdx.x; t <= a.borders; t += N) {
		const int from = t == 0 ? 0 : border[t - 1], to = t < a.borders ? border[t] : a.reach + 1, behind = a.first_behind + a.step_behind * t, ahead = a.first_ahead + a.step_ahead * t;
		put(from, to, behind, ahead);
	}
}
__device__ __forceinline__ int limited(int64_t rel, int reach) { return rel < -reach ? -reach : rel > reach ? reach : (int)rel; }
// the difference of two positions, limited where it passes 64 bits
__device__ __forceinline__ int64_t apart(int64_t k, int64_t q) {
	int64_t d;
	if(__builtin_sub_overflow(k, q, &d)) d = k < q ? INT64_MIN : INT64_MAX;
	return d;
}

// offsets (limited to +-reach) of the E keys of a column chunk from one query
template <int E>
struct keys_of_chunk {
	int64_t k[E];
	int64_t first;
	bool    given;
	__device__ __forceinline__ keys_of_chunk(const args& a, int64_t col) : first(col), given(a.k_pos != nullptr) {
#pragma unroll
		for(int e = 0; e < E; e++) k[e] = given ? a.k_pos[col + e < a.Lk ? col + e : a.Lk - 1] : col + e;
	}
	__device__ __forceinline__ void offsets(int64_t q, int reach, int (&rel)[E]) const {
		if(given) {
#pragma unroll
			for(int e = 0; e < E; e++) rel[e] = limited(apart(k[e], q), reach);
		} else {   // (counted positions: the first one's offset, then one more each)
			const int64_t r0 = apart(first, q);
			const int     low = -reach - E, from = r0 < low ? low : r0 > reach ? reach : (int)r0;
#pragma unroll
			for(int e = 0; e < E; e++) rel[e] = from + e < -reach ? -reach : from + e > reach ? reach : from + e;
		}
	}
};

template <typename T, bool LUT>
__global__ void __launch_bounds__(THREADS) position_bias_kernel(args a) {
	constexpr int E = kind<T>::E;
	__shared__ T   values[LUT ? MAX_OFFSETS : MAX_BUCKETS];   // of the offsets, or of the buckets
	__shared__ int border[MAX_BUCKETS];
	const int64_t  h = blockIdx.z;
	for(int i = threadIdx.x; i < a.borders; i += THREADS) border[i] = border_of(a, i);
	__syncthreads();
	const T* const table = static_cast<const T*>(a.table) + h * a.table_stride[1];
	if constexpr(LUT) {
		for_all_offsets<THREADS>(a, border, [&](int from, int to, int behind, int ahead) {
			const T at_or_behind = table[behind * a.table_stride[0]], in_front = table[ahead * a.table_stride[0]];
			for(int d = from; d < to; d++) {
				values[a.reach - d] = at_or_behind;
				if(d) values[a.reach + d] = in_front;
			}
		});
	} else {
		for(int i = threadIdx.x; i < a.buckets; i += THREADS) values[i] = table[i * a.table_stride[0]];
	}
	__syncthreads();

	const int     columns = 1 << a.columns_log2, tx = threadIdx.x & (columns - 1), ty = threadIdx.x >> a.columns_log2;
	const int64_t col = ((int64_t)blockIdx.x * columns + tx) * E;
	if(col >= a.Lk) return;
	const keys_of_chunk<E> keys(a, col);
	const int64_t row0 = (int64_t)blockIdx.y * a.rows, last = row0 + a.rows < a.Lq ? row0 + a.rows : a.Lq;
	T* const      out = static_cast<T*>(a.out) + h * a.Lq * a.Lk + col;
	const int step = THREADS >> a.columns_log2;
	int64_t   next = a.q_pos && row0 + ty < last ? a.q_pos[row0 + ty] : 0;   // (a row ahead)
	for(int64_t row = row0 + ty; row < last; row += step) {
		int           rel[E];
		const int64_t q = a.q_pos ? next : row + a.q_offset;
		if(a.q_pos && row + step < last) next = a.q_pos[row + step];
		keys.offsets(q, a.reach, rel);
		T v[E];
#pragma unroll
		for(int e = 0; e < E; e++) v[e] = values[LUT ? rel[e] + a.reach : bucket_of(a, border, rel[e])];
		T* const at = out + row * a.Lk;
		if(col + E <= a.Lk) {
			u32x4 packed;
#pragma unroll
			for(int i = 0; i < 4; i++) {
				if constexpr(sizeof(T) == 2) packed[i] = (uint32_t)v[2 * i] | (uint32_t)v[2 * i + 1] << 16;
				else packed[i] = __float_as_uint(v[i]);
			}
			store16(at, packed);
		} else {
#pragma unroll
			for(int e = 0; e < E; e++)
				if(col + e < a.Lk) at[e] = v[e];
		}
	}
}

// Sums by bucket.  Every thread has a column of the bins in LDS to itself (64 threads to a workgroup), so that nothing is added in an order that
// changes; the sums of the threads, then of the workgroups (in 64 bits) follow in a fixed order.  A workgroup's own are in 32 bits, which LDS adds by itself: a thread has 4096 pieces
// at most.
constexpr int COLUMNS = 64;
template <typename T, bool LUT>
__global__ void __launch_bounds__(COLUMNS) position_bias_sums_kernel(args a) {
	constexpr int E = kind<T>::E;
	// (as much LDS as the call needs: with room for the most of everything five workgroups of 65 buckets stood on a compute unit instead of nine)
	extern __shared__ float bins[];   // [buckets][COLUMNS]
	int* const      border = reinterpret_cast<int*>(bins + a.buckets * COLUMNS);         // [borders]
	uint16_t* const bucket = reinterpret_cast<uint16_t*>(border + a.borders);            // [2 reach + 1], where they are tabulated
	const int64_t  z = blockIdx.z, h = z < a.H ? z : z - a.H;   // (the second H of them add up `rest`)
	for(int i = threadIdx.x; i < a.borders; i += COLUMNS) border[i] = border_of(a, i);
	for(int i = 0; i < a.buckets; i++) bins[i * COLUMNS + threadIdx.x] = 0.f;
	__syncthreads();
	if constexpr(LUT)
		for_all_offsets<COLUMNS>(a, border, [&](int from, int to, int behind, int ahead) {
			for(int d = from; d < to; d++) {
				bucket[a.reach - d] = (uint16_t)behind;
				if(d) bucket[a.reach + d] = (uint16_t)ahead;
			}
		});
	__syncthreads();

	const int     columns = 1 << a.columns_log2, tx = threadIdx.x & (columns - 1), ty = threadIdx.x >> a.columns_log2, step = COLUMNS >> a.columns_log2;
	const int64_t col = ((int64_t)blockIdx.x * columns + tx) * E;
	if(col < a.Lk) {
		// Four rows on their way while four are added up.  (Not more: a row's additions are 3 KB of code, which every compute unit has to fetch for some
		// microseconds of work.)
		constexpr int ROWS = 4;
		const keys_of_chunk<E> keys(a, col);
		const int64_t row0 = (int64_t)blockIdx.y * a.rows, last = row0 + a.rows < a.Lq ? row0 + a.rows : a.Lq;
		const T* const grad = static_cast<const T*>(z < a.H ? a.grad : a.rest) + h * a.grad_stride[0] + col;
		const bool     full = col + E <= a.Lk;
		// (an addition that LDS does by itself: nothing waits for the sum so far.  The column is this thread's alone, so the order is the program's)
		auto add = [&](int bk, float v) { __builtin_amdgcn_ds_faddf((__attribute__((address_space(3))) float*)(bins + bk * COLUMNS + threadIdx.x), v, 0, 0, false); };
		struct rows_of {
			u32x4   x[ROWS];
			int64_t q[ROWS];
		};
		auto fetch = [&](rows_of& to, int64_t first) {
#pragma unroll
			for(int i = 0; i < ROWS; i++) {
				const int64_t  row = first + i * step < last ? first + i * step : row0;
				const T* const at  = grad + row * a.grad_stride[1];
				if(full) to.x[i] = load16(at);
				else to.x[i] = cross::load_guarded(at, 0, (int)(a.Lk - col));
				to.q[i] = a.q_pos ? a.q_pos[row] : row + a.q_offset;
			}
		};
		rows_of mine, coming;
		fetch(coming, row0 + ty);
#pragma unroll 1
		for(int64_t first = row0 + ty; first < last; first += ROWS * step) {
			mine = coming;
			if(first + ROWS * step < last) fetch(coming, first + ROWS * step);
#pragma unroll
			for(int i = 0; i < ROWS; i++) {
				if(first + i * step >= last) break;
				int rel[E], bk[E];
				keys.offsets(mine.q[i], a.reach, rel);
#pragma unroll
				for(int e = 0; e < E; e++) bk[e] = LUT ? bucket[rel[e] + a.reach] : bucket_of(a, border, rel[e]);
				bool same = true;
#pragma unroll
				for(int e = 1; e < E; e++) same = same && bk[e] == bk[0];
				if(same) {
					float sum = kind<T>::at(mine.x[i], 0);
#pragma unroll
					for(int e = 1; e < E; e++) sum += kind<T>::at(mine.x[i], e);
					add(bk[0], sum);
				} else {
#pragma unroll
					for(int e = 0; e < E; e++) add(bk[e], kind<T>::at(mine.x[i], e));
				}
			}
		}
	}
	__syncthreads();
	const int64_t part = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, parts = (int64_t)gridDim.x * gridDim.y;
	// a bucket per thread; the threads begin with different columns, which are different banks
	for(int i = threadIdx.x; i < a.buckets; i += COLUMNS) {
		float sum = 0.f;
#pragma unroll 16
		for(int c = 0; c < COLUMNS; c++) sum += bins[i * COLUMNS + ((c + threadIdx.x) & (COLUMNS - 1))];
		a.partial[(z * parts + part) * a.buckets + i] = sum;
	}
}
template <typename T>
__global__ void __launch_bounds__(THREADS) position_bias_join_kernel(args a, int64_t parts) {   // one wavefront per head and bucket
	const int64_t n = (int64_t)blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6);
	const int     lane = threadIdx.x & 63;
	if(n >= a.H * a.buckets) return;
	const int64_t h = n / a.buckets, i = n % a.buckets;
	auto total = [&](const float* of) {
		double sum = 0.0;
		for(int64_t part = lane; part < parts; part += 64) sum += (double)of[(h * parts + part) * a.buckets + i];
#pragma unroll
		for(int k = 32; k; k >>= 1) sum += __shfl_xor(sum, k);
		return sum;
	};
	const double sum   = total(a.partial);
	T            value = kind<T>::bits((float)sum);
	if(a.rest) {   // what a call without rest misses: its answer is `value`
		const double rest = total(a.partial + a.H * parts * a.buckets);
		const float  own  = kind<T>::value(value);
		value = kind<T>::bits(__builtin_isfinite(own) ? (float)(sum + rest - (double)own) : 0.f);
	}
	if(lane == 0) static_cast<T*>(a.out)[i * a.table_stride[0] + h * a.table_stride[1]] = value;
}

// ---- host side -------------------------------------------------------------------------------------------------------------
// whole numbers of any length in digits of 32 bits, lowest first: products of at most MAX_BUCKETS factors
struct whole {
	int      n = 1;
	uint32_t digit[MAX_BUCKETS + 1] = {1u};
	void times(uint32_t f) {
		uint64_t carry = 0;
		for(int i = 0; i < n; i++) carry += (uint64_t)digit[i] * f, digit[i] = (uint32_t)carry, carry >>= 32;
		if(carry) digit[n++] = (uint32_t)carry;
	}
	bool not_less(const whole& b) const {
		if(n != b.n) return n > b.n;
		for(int i = n - 1; i >= 0; i--)
			if(digit[i] != b.digit[i]) return digit[i] > b.digit[i];
		return true;
	}
};
// d^far >= r^i near^(far - i)
bool reaches(uint32_t d, uint32_t r, uint32_t near, int i, int far) {
	whole a, b;
	for(int k = 0; k < far; k++) a.times(d), b.times(k < i ? r : near);
	return a.not_less(b);
}

// The borders of a set of settings take microseconds to work out; a thread keeps those of its last one.
struct worked_out {
	int64_t buckets = 0, max_distance = 0;
	int32_t both = 0, border[MAX_BUCKETS / 2];
};
// the borders behind the first near, n - 1 - near of them
void log_borders(int64_t buckets, int64_t max_distance, bool both, int32_t* border) {
	static thread_local worked_out last;
	const int n = (int)(both ? buckets / 2 : buckets), near = n / 2, far = n - near;
	if(last.buckets != buckets || last.max_distance != max_distance || last.both != both) {
		for(int i = 1; i < far; i++) {   // the smallest d with (d / near)^far >= (max_distance / near)^i
			const long double y = near * powl((long double)max_distance / near, (long double)i / far), r = roundl(y);
			int               d;
			if(fabsl(y - r) > 1e-6L) d = (int)ceill(y);
			else d = (int)r + (reaches((uint32_t)r, (uint32_t)max_distance, (uint32_t)near, i, far) ? 0 : 1);
			last.border[i - 1] = d;
		}
		last.buckets = buckets, last.max_distance = max_distance, last.both = both;
	}
	for(int i = 0; i < far - 1; i++) border[i] = last.border[i];
}

int prepare(const af3_position_bias_params* p, args& a) {
	if(!p) return AF3_ERR_NULL_POINTER;
	if(p->dtype != AF3_F32 && p->dtype != AF3_BF16) return AF3_ERR_BAD_DTYPE;
	if(p->buckets <= 0 || p->buckets > MAX_BUCKETS || p->H <= 0 || p->H > 0xffff || p->Lq <= 0 || p->Lk <= 0 || p->Lq > 0x3fffffff || p->Lk > 0x3fffffff) return AF3_ERR_BAD_SHAPE;
	if(p->table_stride[0] < 0 || p->table_stride[1] < 0) return AF3_ERR_BAD_STRIDE;
	if(p->max_distance < 1 || p->max_distance > 0x3fffffff || p->q_offset > (int64_t)1 << 62 || p->q_offset < -((int64_t)1 << 62)) return AF3_ERR_BAD_ARGUMENT;
	const bool both = p->bidirectional != 0;
	a.buckets = (int)p->buckets;
	if(p->scheme == AF3_POSITION_CLIP) {
		if(p->buckets != p->max_distance * (both ? 2 : 1) + 1) return AF3_ERR_BAD_ARGUMENT;
		a.borders = (int)p->max_distance;
		a.near = a.borders;
		a.first_behind = both ? a.borders : 0, a.step_behind = 1, a.first_ahead = both ? a.borders : 0, a.step_ahead = both ? -1 : 0;
	} else if(p->scheme == AF3_POSITION_LOG) {
		if(both && p->buckets % 2 != 0) return AF3_ERR_BAD_ARGUMENT;
		const int n = (int)(both ? p->buckets / 2 : p->buckets), near = n / 2;
		if(near < 1 || p->max_distance <= near) return AF3_ERR_BAD_ARGUMENT;
		a.borders = n - 1;
		a.near = near;
		log_borders(p->buckets, p->max_distance, both, a.far_border);
		a.first_behind = 0, a.step_behind = 1, a.first_ahead = both ? n : 0, a.step_ahead = both ? 1 : 0;
	} else {
		return AF3_ERR_BAD_ARGUMENT;
	}
	a.reach = a.borders == a.near ? a.near : a.far_border[a.borders - a.near - 1];
	a.q_pos = p->q_positions, a.k_pos = p->k_positions, a.q_offset = p->q_offset;
	a.table_stride[0] = p->table_stride[0], a.table_stride[1] = p->table_stride[1];
	a.grad_stride[0] = p->grad_stride[0], a.grad_stride[1] = p->grad_stride[1];
	a.H = p->H, a.Lq = p->Lq, a.Lk = p->Lk;
	a.table = p->table, a.out = p->out, a.grad = p->grad, a.rest = p->grad_residual, a.partial = nullptr;
	return AF3_OK;
}
bool tabulated(const args& a) { return 2 * (int64_t)a.reach + 1 <= MAX_OFFSETS; }

// columns and rows of a workgroup of n threads, and the grid: about `each` 16-byte pieces per thread
dim3 shape(args& a, int E, int n, int64_t each) {
	const int64_t chunks = (a.Lk + E - 1) / E;
	a.columns_log2 = 0;
	while((1 << a.columns_log2) < n && (1 << a.columns_log2) < chunks) a.columns_log2++;
	const int64_t across = (chunks + (1 << a.columns_log2) - 1) >> a.columns_log2, deep = n >> a.columns_log2;
	int64_t       rows = deep * each;
	while((a.Lq + rows - 1) / rows > 0xffff) rows *= 2;
	a.rows = (int32_t)(rows < a.Lq ? rows : a.Lq);
	return dim3((uint32_t)across, (uint32_t)((a.Lq + a.rows - 1) / a.rows), (uint32_t)a.H);
}
dim3 sums_shape(args& a, int E) {
	// about 2048 workgroups, of 8 pieces per thread at least: each clears its bins and adds them up, whatever it reads (16 x 768 x 768 in fp32 takes 23.5 us with 3 buckets,
	// 28 with 65, 49 with 129)
	const int64_t pieces = a.H * a.Lq * ((a.Lk + E - 1) / E);
	int64_t       each = pieces / (2048 * COLUMNS);
	dim3 grid = shape(a, E, COLUMNS, each < 8 ? 8 : each > 4096 ? 4096 : each);
	if(a.rest) grid.z *= 2;   // (cut like the call without it, whose sums these have to be to the bit)
	return grid;
}
dim3 forward_shape(args& a, int E) {
	// about 1024 workgroups, of one to 16 pieces per thread
	const int64_t each = a.H * a.Lq * ((a.Lk + E - 1) / E) / (1024 * THREADS);
	return shape(a, E, THREADS, each < 1 ? 1 : each > 16 ? 16 : each);
}

template <typename T>
int forward(const args& a, dim3 grid, hipStream_t s) {
	if(tabulated(a)) hipLaunchKernelGGL((position_bias_kernel<T, true>), grid, dim3(THREADS), 0, s, a);
	else hipLaunchKernelGGL((position_bias_kernel<T, false>), grid, dim3(THREADS), 0, s, a);
	return launch_status();
}
template <typename T, bool LUT>
int sums(const args& a, dim3 grid, hipStream_t s) {
	const int lds = a.buckets * COLUMNS * 4 + a.borders * 4 + (LUT ? (2 * a.reach + 1) * 2 : 0);
	if(lds > 32768 && hipFuncSetAttribute(reinterpret_cast<const void*>(&position_bias_sums_kernel<T, LUT>), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
		(void)hipGetLastError();
		return AF3_ERR_LAUNCH;
	}
	hipLaunchKernelGGL((position_bias_sums_kernel<T, LUT>), grid, dim3(COLUMNS), lds, s, a);
	return launch_status();
}
template <typename T>
int backward(const args& a, dim3 grid, hipStream_t s) {
	if(const int rc = tabulated(a) ? sums<T, true>(a, grid, s) : sums<T, false>(a, grid, s); rc != AF3_OK) return rc;
	hipLaunchKernelGGL(position_bias_join_kernel<T>, dim3((uint32_t)((a.H * a.buckets + 3) / 4)), dim3(THREADS), 0, s, a, (int64_t)grid.x * grid.y);
	return launch_status();
}

}  // namespace position
}  // namespace af3

using namespace af3;

extern "C" int af3_position_bias_forward(const af3_position_bias_params* params, void* hip_stream) {
	position::args a;
	if(const int rc = position::prepare(params, a); rc != AF3_OK) return rc;
	if(!params->table || !params->out) return AF3_ERR_NULL_POINTER;
	if(const int dc = current_device_status(); dc != AF3_OK) return dc;
	const hipStream_t s = static_cast<hipStream_t>(hip_stream);
	const dim3 grid = position::forward_shape(a, params->dtype == AF3_F32 ? 4 : 8);
	return params->dtype == AF3_F32 ? position::forward<float>(a, grid, s) : position::forward<uint16_t>(a, grid, s);
}

extern "C" int64_t af3_position_bias_workspace_bytes(const af3_position_bias_params* params) {
	position::args a;
	if(const int rc = position::prepare(params, a); rc != AF3_OK) return rc;
	if(a.rest && a.H > 0x7fff) return AF3_ERR_BAD_SHAPE;
	const dim3 grid = position::sums_shape(a, params->dtype == AF3_F32 ? 4 : 8);
	return (int64_t)grid.x * grid.y * grid.z * a.buckets * 4;
}

extern "C" int af3_position_bias_backward(const af3_position_bias_params* params, void* hip_stream) {
	position::args a;
	if(const int rc = position::prepare(params, a); rc != AF3_OK) return rc;
	if(!params->grad || !params->out || !params->workspace) return AF3_ERR_NULL_POINTER;
	if(a.rest && a.H > 0x7fff) return AF3_ERR_BAD_SHAPE;
	if(params->grad_stride[0] < 0 || params->grad_stride[1] < 0) return AF3_ERR_BAD_STRIDE;
	if((params->buckets > 1 && params->table_stride[0] == 0) || (params->H > 1 && params->table_stride[1] == 0)) return AF3_ERR_BAD_STRIDE;   // (results may not share a place)
	const dim3 grid = position::sums_shape(a, params->dtype == AF3_F32 ? 4 : 8);
	if(params->workspace_bytes < (int64_t)grid.x * grid.y * grid.z * a.buckets * 4 || (reinterpret_cast<uintptr_t>(params->workspace) & 15)) return AF3_ERR_BAD_ARGUMENT;
	if(const int dc = current_device_status(); dc != AF3_OK) return dc;
	a.partial = static_cast<float*>(params->workspace);
	const hipStream_t s = static_cast<hipStream_t>(hip_stream);
	return params->dtype == AF3_F32 ? position::backward<float>(a, grid, s) : position::backward<uint16_t>(a, grid, s);
}
