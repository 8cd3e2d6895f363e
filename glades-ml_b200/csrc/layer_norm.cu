// Layer norm of a [rows][n] matrix, forward and backward.
//     mu = sum(x) / n,  v = sum((x - mu)^2) / n,  r = 1 / sqrt(v + eps),  xh = (x - mu) r,  y = gain xh + shift
//     g = gain dy,  dx = r (g - sum(g) / n - xh sum(g xh) / n),  dgain = sum_rows dy xh,  dshift = sum_rows dy
// Bound: HBM.  Forward reads x and writes y once, backward reads x and dy and writes dx once.
// A row is held in registers by a group of lanes, so that its statistics cost no second read: the variance is the mean of
// (x - mu)^2, not a difference of two large sums.  Everything between the loads and the stores is fp32, each result is
// rounded to the tensors' type once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "internal.h"

namespace glb {
namespace {

constexpr int LN_SMS = 148;
constexpr int LN_THREADS = 256;     // threads of a CTA that holds several groups
constexpr int LN_GROUP_MAX = 512;   // lanes of the largest group
constexpr int LN_ELEMS = 16;        // values of a row that a lane holds
constexpr int LN_ELEMS_LONG = 32;   // forward, rows too long for 512 lanes of 16

// VEC neighbouring values of type T as one load or store
template <int BYTES> struct Word;
template <> struct Word<2> { typedef unsigned short type; };
template <> struct Word<4> { typedef unsigned type; };
template <> struct Word<16> { typedef uint4 type; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T, int VEC>
struct Pack
{
	typename Word<sizeof(T) * VEC>::type w;
	__device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const decltype(w)*>(p); }
	__device__ __forceinline__ void store(T* p) const { *reinterpret_cast<decltype(w)*>(p) = w; }
	__device__ __forceinline__ float get(int i) const { return to_float(reinterpret_cast<const T*>(&w)[i]); }
	__device__ __forceinline__ void set(int i, float v) { reinterpret_cast<T*>(&w)[i] = from_float<T>(v); }
};

// The lanes that share a row.  Groups of at most 32 lanes (a power of two) lie in one warp; larger ones are whole warps of one
// CTA and meet at a barrier of their own (number 1 + group), their sums in `slot`.
struct Group
{
	int size, lane, index;
	float2* slot;  // [2][warps of the group], written in turn
	int turn;
	__device__ Group(int size_, float2* shared) : size(size_), turn(0)
	{
		index = (int)threadIdx.x / size;
		lane = (int)threadIdx.x - index * size;
		slot = shared + index * 2 * ((size + 31) / 32);
	}
	// the two sums over the group, on every lane, added in the same order whatever lane asks
	template <bool WIDE>
	__device__ __forceinline__ float2 sum(float a, float b)
	{
		if constexpr (!WIDE)
		{
			for (int o = size >> 1; o > 0; o >>= 1)
			{
				a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
				b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
			}
			return make_float2(a, b);
		}
		else
		{
#pragma unroll
			for (int o = 16; o > 0; o >>= 1)
			{
				a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
				b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
			}
			const int warps = size >> 5;
			float2* s = slot + turn * warps;
			turn ^= 1;
			if ((lane & 31) == 0) s[lane >> 5] = make_float2(a, b);
			asm volatile("bar.sync %0, %1;" ::"r"(1 + index), "r"(size) : "memory");
			const float2 v = (lane & 15) < warps ? s[lane & 15] : make_float2(0.0f, 0.0f);  // at most 16 warps: both half warps add them
			a = v.x;
			b = v.y;
#pragma unroll
			for (int o = 8; o > 0; o >>= 1)
			{
				a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
				b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
			}
			return make_float2(a, b);
		}
	}
};

// ---- forward -------------------------------------------------------------------------------------------------
// Groups walk the rows; a row's values are asked for before the row in front is worked on (the loads of one row alone leave
// HBM idle for as long as its sums take).  Gain and shift stay in registers.
template <class T, int VEC, int ELEMS, bool WIDE>
__global__ void __launch_bounds__(LN_GROUP_MAX) norm_kernel(const LayerNormArgs p, int group)
{
	constexpr int V = ELEMS / VEC;
	constexpr bool KEEP = ELEMS == LN_ELEMS;
	__shared__ float2 slots[2 * LN_GROUP_MAX / 32];
	Group gr(group, slots);
	const int groups = blockDim.x / group;
	const long long step = (long long)gridDim.x * groups;
	const T* X = static_cast<const T*>(p.x);
	T* Y = static_cast<T*>(p.y);
	const float inv_n = 1.0f / (float)p.n;
	float gain[KEEP ? ELEMS : 1], shift[KEEP ? ELEMS : 1];
	if (KEEP)
	{
#pragma unroll
		for (int v = 0; v < V; ++v)
#pragma unroll
			for (int i = 0; i < VEC; ++i)
			{
				const int c = (v * group + gr.lane) * VEC + i;
				gain[v * VEC + i] = p.gain && c < p.n ? p.gain[c] : 1.0f;
				shift[v * VEC + i] = p.shift && c < p.n ? p.shift[c] : 0.0f;
			}
	}
	auto fetch = [&](long long row, Pack<T, VEC>(&a)[V]) {
#pragma unroll
		for (int v = 0; v < V; ++v)
		{
			const int c = (v * group + gr.lane) * VEC;
			if (row < p.rows && c < p.n) a[v].load(X + row * p.ldx + c);
		}
	};
	long long row = (long long)blockIdx.x * groups + gr.index;
	Pack<T, VEC> next[V];
	fetch(row, next);
	// (every group of a warp walks as often as the warp's first, whose row is the smallest: the shuffles need all lanes)
	const long long walk = WIDE ? row : (long long)blockIdx.x * groups + ((int)threadIdx.x & ~31) / group;
	for (long long first = walk; first < p.rows; first += step, row += step)
	{
		float x[ELEMS];
		float s = 0.0f;
#pragma unroll
		for (int v = 0; v < V; ++v)
#pragma unroll
			for (int i = 0; i < VEC; ++i)
			{
				const bool in = row < p.rows && (v * group + gr.lane) * VEC < p.n;
				x[v * VEC + i] = in ? next[v].get(i) : 0.0f;
				s += x[v * VEC + i];
			}
		fetch(row + step, next);
		const float mean = gr.sum<WIDE>(s, 0.0f).x / (float)p.n;  // (a division: a row of equal values keeps its mean)
		float q = 0.0f;
#pragma unroll
		for (int v = 0; v < V; ++v)
#pragma unroll
			for (int i = 0; i < VEC; ++i)
				if ((v * group + gr.lane) * VEC < p.n)
				{
					const float d = x[v * VEC + i] - mean;
					q = fmaf(d, d, q);
				}
		const float rstd = 1.0f / sqrtf(gr.sum<WIDE>(q, 0.0f).x * inv_n + p.eps);
		if (row >= p.rows) continue;
#pragma unroll
		for (int v = 0; v < V; ++v)
		{
			const int c = (v * group + gr.lane) * VEC;
			if (c >= p.n) continue;
			Pack<T, VEC> o;
#pragma unroll
			for (int i = 0; i < VEC; ++i)
			{
				const float ga = KEEP ? gain[KEEP ? v * VEC + i : 0] : (p.gain ? p.gain[c + i] : 1.0f);
				const float sh = KEEP ? shift[KEEP ? v * VEC + i : 0] : (p.shift ? p.shift[c + i] : 0.0f);
				o.set(i, fmaf((x[v * VEC + i] - mean) * rstd, ga, sh));
			}
			o.store(Y + row * p.ldy + c);
		}
		if (gr.lane == 0)
		{
			if (p.mean) p.mean[row] = mean;
			if (p.rstd) p.rstd[row] = rstd;
		}
	}
}

// Rows too long for a group's registers: one CTA per row reads it three times (the second and third time from L2).
template <class T>
__global__ void __launch_bounds__(LN_GROUP_MAX) norm_long_kernel(const LayerNormArgs p)
{
	__shared__ float2 slots[2 * LN_GROUP_MAX / 32];
	Group gr(LN_GROUP_MAX, slots);
	const float inv_n = 1.0f / (float)p.n;
	for (long long row = blockIdx.x; row < p.rows; row += gridDim.x)
	{
		const T* x = static_cast<const T*>(p.x) + row * p.ldx;
		T* y = static_cast<T*>(p.y) + row * p.ldy;
		float s = 0.0f;
		for (long long c = threadIdx.x; c < p.n; c += LN_GROUP_MAX) s += to_float(x[c]);
		const float mean = gr.sum<true>(s, 0.0f).x / (float)p.n;
		float q = 0.0f;
		for (long long c = threadIdx.x; c < p.n; c += LN_GROUP_MAX)
		{
			const float d = to_float(x[c]) - mean;
			q = fmaf(d, d, q);
		}
		const float rstd = 1.0f / sqrtf(gr.sum<true>(q, 0.0f).x * inv_n + p.eps);
		for (long long c = threadIdx.x; c < p.n; c += LN_GROUP_MAX)
			y[c] = from_float<T>(fmaf((to_float(x[c]) - mean) * rstd, p.gain ? p.gain[c] : 1.0f, p.shift ? p.shift[c] : 0.0f));
		if (threadIdx.x == 0)
		{
			if (p.mean) p.mean[row] = mean;
			if (p.rstd) p.rstd[row] = rstd;
		}
	}
}

// ---- backward ------------------------------------------------------------------------------------------------
// The same groups; both row sums in one exchange.  A lane keeps the same columns for all its rows and adds their dgain and
// dshift up in registers; a CTA's groups are added in a fixed order and leave as one partial row, which norm_columns_kernel
// adds up: no atomics, two runs give the same bits.
template <class T, int VEC, bool WIDE>
__global__ void __launch_bounds__(LN_GROUP_MAX) norm_backward_kernel(const LayerNormArgs p, int group)
{
	constexpr int ELEMS = LN_ELEMS, V = ELEMS / VEC;
	extern __shared__ float2 sums[];  // [groups or (in-warp groups) warps][n]
	__shared__ float2 slots[2 * LN_GROUP_MAX / 32];
	Group gr(group, slots);
	const int groups = blockDim.x / group;
	const long long step = (long long)gridDim.x * groups;
	const T* X = static_cast<const T*>(p.x);
	const T* DY = static_cast<const T*>(p.dy);
	T* DX = static_cast<T*>(p.dx);
	const float inv_n = 1.0f / (float)p.n;
	float gain[ELEMS], dg[ELEMS], ds[ELEMS];
#pragma unroll
	for (int v = 0; v < V; ++v)
#pragma unroll
		for (int i = 0; i < VEC; ++i)
		{
			const int c = (v * group + gr.lane) * VEC + i;
			gain[v * VEC + i] = p.gain && c < p.n ? p.gain[c] : 1.0f;
			dg[v * VEC + i] = ds[v * VEC + i] = 0.0f;
		}
	Pack<T, VEC> xn[V], dn[V];
	float mean_n = 0.0f, rstd_n = 0.0f;
	auto fetch = [&](long long row) {
		if (row >= p.rows) return;
		mean_n = p.mean[row];
		rstd_n = p.rstd[row];
#pragma unroll
		for (int v = 0; v < V; ++v)
		{
			const int c = (v * group + gr.lane) * VEC;
			if (c < p.n)
			{
				xn[v].load(X + row * p.ldx + c);
				dn[v].load(DY + row * p.lddy + c);
			}
		}
	};
	long long row = (long long)blockIdx.x * groups + gr.index;
	fetch(row);
	const long long walk = WIDE ? row : (long long)blockIdx.x * groups + ((int)threadIdx.x & ~31) / group;
	for (long long first = walk; first < p.rows; first += step, row += step)
	{
		float xh[ELEMS], dy[ELEMS];
		const float mean = mean_n, rstd = rstd_n;
		float a = 0.0f, b = 0.0f;
#pragma unroll
		for (int v = 0; v < V; ++v)
#pragma unroll
			for (int i = 0; i < VEC; ++i)
			{
				const int e = v * VEC + i;
				const bool in = row < p.rows && (v * group + gr.lane) * VEC < p.n;
				xh[e] = in ? (xn[v].get(i) - mean) * rstd : 0.0f;
				dy[e] = in ? dn[v].get(i) : 0.0f;
				const float g = dy[e] * gain[e];
				a += g;
				b = fmaf(g, xh[e], b);
				dg[e] = fmaf(dy[e], xh[e], dg[e]);
				ds[e] += dy[e];
			}
		fetch(row + step);
		const float2 s = gr.sum<WIDE>(a, b);
		const float ma = s.x * inv_n, mb = s.y * inv_n;
		if (!DX || row >= p.rows) continue;
#pragma unroll
		for (int v = 0; v < V; ++v)
		{
			const int c = (v * group + gr.lane) * VEC;
			if (c >= p.n) continue;
			Pack<T, VEC> o;
#pragma unroll
			for (int i = 0; i < VEC; ++i)
			{
				const int e = v * VEC + i;
				o.set(i, rstd * (fmaf(dy[e], gain[e], -ma) - xh[e] * mb));
			}
			o.store(DX + row * p.lddx + c);
		}
	}
	if (!p.part) return;
	if (!WIDE)
	{
		// the warp's groups hold the same columns on lanes that are a group apart
#pragma unroll
		for (int e = 0; e < ELEMS; ++e)
			for (int o = group; o < 32; o <<= 1)
			{
				dg[e] += __shfl_xor_sync(0xFFFFFFFFu, dg[e], o);
				ds[e] += __shfl_xor_sync(0xFFFFFFFFu, ds[e], o);
			}
	}
	const int parts = WIDE ? groups : (int)blockDim.x / 32;
	const int part = WIDE ? gr.index : (int)threadIdx.x / 32;
	if (WIDE || (int)(threadIdx.x & 31) < group)
	{
#pragma unroll
		for (int v = 0; v < V; ++v)
#pragma unroll
			for (int i = 0; i < VEC; ++i)
			{
				const int c = (v * group + gr.lane) * VEC + i;
				if (c >= p.n) continue;
				if (parts == 1) p.part[(long long)blockIdx.x * p.n + c] = make_float2(dg[v * VEC + i], ds[v * VEC + i]);
				else sums[(long long)part * p.n + c] = make_float2(dg[v * VEC + i], ds[v * VEC + i]);
			}
	}
	if (parts == 1) return;
	__syncthreads();
	for (int c = threadIdx.x; c < p.n; c += blockDim.x)
	{
		float2 t = sums[c];
		for (int k = 1; k < parts; ++k)
		{
			t.x += sums[k * p.n + c].x;
			t.y += sums[k * p.n + c].y;
		}
		p.part[(long long)blockIdx.x * p.n + c] = t;
	}
}

// Long rows: dx by a CTA per row in two passes ...
template <class T>
__global__ void __launch_bounds__(LN_GROUP_MAX) norm_backward_long_kernel(const LayerNormArgs p)
{
	__shared__ float2 slots[2 * LN_GROUP_MAX / 32];
	Group gr(LN_GROUP_MAX, slots);
	const float inv_n = 1.0f / (float)p.n;
	for (long long row = blockIdx.x; row < p.rows; row += gridDim.x)
	{
		const T* x = static_cast<const T*>(p.x) + row * p.ldx;
		const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
		T* dx = static_cast<T*>(p.dx) + row * p.lddx;
		const float mean = p.mean[row], rstd = p.rstd[row];
		float a = 0.0f, b = 0.0f;
		for (long long c = threadIdx.x; c < p.n; c += LN_GROUP_MAX)
		{
			const float g = to_float(dy[c]) * (p.gain ? p.gain[c] : 1.0f);
			a += g;
			b = fmaf(g, (to_float(x[c]) - mean) * rstd, b);
		}
		const float2 s = gr.sum<true>(a, b);
		const float ma = s.x * inv_n, mb = s.y * inv_n;
		for (long long c = threadIdx.x; c < p.n; c += LN_GROUP_MAX)
			dx[c] = from_float<T>(rstd * (fmaf(to_float(dy[c]), p.gain ? p.gain[c] : 1.0f, -ma) - (to_float(x[c]) - mean) * rstd * mb));
	}
}
// ... and the columns' sums over a slice of the rows
template <class T>
__global__ void __launch_bounds__(LN_THREADS) norm_slices_kernel(const LayerNormArgs p, int slices)
{
	const long long c = (long long)blockIdx.x * LN_THREADS + threadIdx.x;
	if (c >= p.n) return;
	const T* x = static_cast<const T*>(p.x);
	const T* dy = static_cast<const T*>(p.dy);
	float2 t = make_float2(0.0f, 0.0f);
	for (long long row = blockIdx.y; row < p.rows; row += slices)
	{
		const float d = to_float(dy[row * p.lddy + c]);
		t.x = fmaf(d, (to_float(x[row * p.ldx + c]) - p.mean[row]) * p.rstd[row], t.x);
		t.y += d;
	}
	p.part[(long long)blockIdx.y * p.n + c] = t;
}

// dgain | dshift from `parts` partial rows: 32 columns per CTA, eight slices of the partials, added in a fixed order
__global__ void __launch_bounds__(LN_THREADS) norm_columns_kernel(const float2* part, int parts, int n, float* dgain, float* dshift)
{
	__shared__ float2 sums[8][33];
	const int k = threadIdx.x & 31, slice = threadIdx.x >> 5;
	const long long c = (long long)blockIdx.x * 32 + k;
	cudaGridDependencySynchronize();
	float2 t = make_float2(0.0f, 0.0f);
	if (c < n)
	{
#pragma unroll 4
		for (int r = slice; r < parts; r += 8)
		{
			const float2 v = part[(long long)r * n + c];
			t.x += v.x;
			t.y += v.y;
		}
	}
	sums[slice][k] = t;
	__syncthreads();
	if (slice != 0 || c >= n) return;
#pragma unroll
	for (int s = 1; s < 8; ++s)
	{
		t.x += sums[s][k].x;
		t.y += sums[s][k].y;
	}
	if (dgain) dgain[c] = t.x;
	if (dshift) dshift[c] = t.y;
}

// ---- a network's training step around them ------------------------------------------------------------------------
__global__ void __launch_bounds__(LN_THREADS) activation_gradient_kernel(float* D, const float* A, long long rows, int n, long long ld, int act, float par)
{
	for (long long r = blockIdx.y; r < rows; r += gridDim.y)
		for (int c = blockIdx.x * LN_THREADS + threadIdx.x; c < n; c += gridDim.x * LN_THREADS) D[r * ld + c] *= act_der_b(A[r * ld + c], act, par);
}
__global__ void __launch_bounds__(LN_THREADS) norm_update_kernel(float* param, int n, float step, int* flags)
{
	const int i = blockIdx.x * LN_THREADS + threadIdx.x;  // gain | shift
	if (i >= 2 * n) return;
	const float v = fmaf(-step, param[2 * (long long)n + i], param[i]);
	param[i] = v;
	if (!isfinite(v)) atomicOr(flags, 1);
}

// ---- host ----------------------------------------------------------------------------------------------------
// Lanes of a row: in one warp a power of two, else whole warps.
int group_lanes(int n, int elems)
{
	const int lanes = (n + elems - 1) / elems;
	if (lanes > 32) return (lanes + 31) / 32 * 32;
	int g = 1;
	while (g < lanes) g *= 2;
	return g;
}
int group_threads(int group) { return group <= LN_THREADS ? group * (LN_THREADS / group) : group; }

// The widest access that every row of every tensor allows: 16 bytes, 4 bytes (16-bit types), one value.
bool aligned(const LayerNormArgs& a, int size, int bytes)
{
	auto ok = [&](const void* p, long long ld) { return !p || ((uintptr_t)p % bytes == 0 && (ld * size) % bytes == 0); };
	return ((long long)a.n * size) % bytes == 0 && ok(a.x, a.ldx) && ok(a.y, a.ldy) && ok(a.dy, a.lddy) && ok(a.dx, a.lddx);
}

// CTAs of the backward kernel, each of which leaves one partial row
int backward_ctas(long long rows, int n)
{
	const int group = group_lanes(n, LN_ELEMS);
	const int groups = group_threads(group) / group;
	const long long want = (rows + groups - 1) / groups;
	const long long most = LN_SMS * 2;
	return (int)(want < most ? want : most);
}
bool backward_long(int n) { return n > LN_GROUP_MAX * LN_ELEMS; }
int backward_slices(long long rows) { return (int)(rows < 32 ? rows : 32); }

template <class T, int VEC>
cudaError_t forward_vec(const LayerNormArgs& a, cudaStream_t s)
{
	const bool lengthy = a.n > LN_GROUP_MAX * LN_ELEMS;
	const int group = group_lanes(a.n, lengthy ? LN_ELEMS_LONG : LN_ELEMS);
	const int threads = group_threads(group);
	const long long want = (a.rows + threads / group - 1) / (threads / group);
	const long long most = (long long)LN_SMS * (2048 / threads);
	const unsigned grid = (unsigned)(want < most ? want : most);
	if (lengthy) norm_kernel<T, VEC, LN_ELEMS_LONG, true><<<grid, threads, 0, s>>>(a, group);
	else if (group > 32) norm_kernel<T, VEC, LN_ELEMS, true><<<grid, threads, 0, s>>>(a, group);
	else norm_kernel<T, VEC, LN_ELEMS, false><<<grid, threads, 0, s>>>(a, group);
	return cudaGetLastError();
}

template <class T, int VEC>
cudaError_t backward_vec(const LayerNormArgs& a, cudaStream_t s)
{
	const int group = group_lanes(a.n, LN_ELEMS);
	const int threads = group_threads(group);
	const int parts = group > 32 ? threads / group : threads / 32;
	const size_t smem = parts > 1 ? (size_t)parts * a.n * sizeof(float2) : 0;
	const int grid = backward_ctas(a.rows, a.n);
	if (group > 32) norm_backward_kernel<T, VEC, true><<<grid, threads, smem, s>>>(a, group);
	else norm_backward_kernel<T, VEC, false><<<grid, threads, smem, s>>>(a, group);
	return cudaGetLastError();
}

template <class T>
cudaError_t forward_type(const LayerNormArgs& a, cudaStream_t s)
{
	if (a.n > LN_GROUP_MAX * LN_ELEMS_LONG)
	{
		const long long most = LN_SMS * 4;
		norm_long_kernel<T><<<(unsigned)(a.rows < most ? a.rows : most), LN_GROUP_MAX, 0, s>>>(a);
		return cudaGetLastError();
	}
	if (aligned(a, sizeof(T), 16)) return forward_vec<T, 16 / sizeof(T)>(a, s);
	if (sizeof(T) == 2 && aligned(a, sizeof(T), 4)) return forward_vec<T, 4 / sizeof(T)>(a, s);
	return forward_vec<T, 1>(a, s);
}

template <class T>
cudaError_t backward_type(const LayerNormArgs& a, cudaStream_t s)
{
	int parts;
	if (backward_long(a.n))
	{
		parts = backward_slices(a.rows);
		if (a.part)
		{
			norm_slices_kernel<T><<<dim3((unsigned)((a.n + LN_THREADS - 1) / LN_THREADS), (unsigned)parts), LN_THREADS, 0, s>>>(a, parts);
			cudaError_t e = cudaGetLastError();
			if (e != cudaSuccess) return e;
		}
		if (a.dx)
		{
			const long long most = LN_SMS * 4;
			norm_backward_long_kernel<T><<<(unsigned)(a.rows < most ? a.rows : most), LN_GROUP_MAX, 0, s>>>(a);
			cudaError_t e = cudaGetLastError();
			if (e != cudaSuccess) return e;
		}
	}
	else
	{
		parts = backward_ctas(a.rows, a.n);
		cudaError_t e;
		if (aligned(a, sizeof(T), 16)) e = backward_vec<T, 16 / sizeof(T)>(a, s);
		else if (sizeof(T) == 2 && aligned(a, sizeof(T), 4)) e = backward_vec<T, 4 / sizeof(T)>(a, s);
		else e = backward_vec<T, 1>(a, s);
		if (e != cudaSuccess) return e;
	}
	if (!a.part) return cudaSuccess;
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned)((a.n + 31) / 32));
	cfg.blockDim = dim3(LN_THREADS);
	cfg.stream = s;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	at[0].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = at;
	cfg.numAttrs = 1;
	return cudaLaunchKernelEx(&cfg, norm_columns_kernel, (const float2*)a.part, parts, a.n, a.dgain, a.dshift);
}

}  // namespace

size_t layer_norm_partial_rows(long long rows, int n)
{
	if (rows < 1) return 0;
	return (size_t)(backward_long(n) ? backward_slices(rows) : backward_ctas(rows, n));
}

cudaError_t launch_layer_norm(const LayerNormArgs& a, int type, cudaStream_t s)
{
	if (type == GL_F32) return forward_type<float>(a, s);
	if (type == GL_BF16) return forward_type<__nv_bfloat16>(a, s);
	return forward_type<__half>(a, s);
}

cudaError_t launch_layer_norm_backward(const LayerNormArgs& a, int type, cudaStream_t s)
{
	if (type == GL_F32) return backward_type<float>(a, s);
	if (type == GL_BF16) return backward_type<__nv_bfloat16>(a, s);
	return backward_type<__half>(a, s);
}

cudaError_t launch_activation_gradient(float* D, const float* A, long long rows, int n, long long ld, int act, float par, cudaStream_t s)
{
	const dim3 grid((unsigned)((n + LN_THREADS - 1) / LN_THREADS), (unsigned)(rows < 4096 ? rows : 4096));
	activation_gradient_kernel<<<grid, LN_THREADS, 0, s>>>(D, A, rows, n, ld, act, par);
	return cudaGetLastError();
}

cudaError_t launch_norm_update(float* param, int n, float step, int* flags, cudaStream_t s)
{
	norm_update_kernel<<<(unsigned)((2 * (long long)n + LN_THREADS - 1) / LN_THREADS), LN_THREADS, 0, s>>>(param, n, step, flags);
	return cudaGetLastError();
}

}  // namespace glb
