// Layer norm of a [rows][n] matrix, forward and backward.
//     mu = sum(x) / n,  v = sum((x - mu)^2) / n,  r = 1 / sqrt(v + eps),  xh = (x - mu) r,  y = gain xh + shift
//     g = gain dy,  dx = r (g - sum(g) / n - xh sum(g xh) / n),  dgain = sum_rows dy xh,  dshift = sum_rows dy
// Bound: HBM.  Forward reads x and writes y once, backward reads x and dy and writes dx once.
// A row is held in registers by a group of lanes, so that its statistics cost no second read: the variance is the mean of
// (x - mu)^2, not a difference of two large sums.  Everything between the loads and the stores is fp32, each result is
// rounded to the tensors' type once.
#include <algorithm>

#include "layer_norm.cuh"
#include "tc_gemm.h"

namespace glb {
namespace {

constexpr int LN_THREADS = 256;     // threads of a CTA that holds several groups
constexpr int LN_GROUP_MAX = 512;   // lanes of the largest group (forward: LN_THREADS)
constexpr int LN_SLICES = 32;       // of the backward pass's partial rows, added side by side
constexpr int LN_ELEMS = 16;        // values of a row that a lane holds in the backward pass

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
	// the sum over the group, on every lane
	template <bool WIDE>
	__device__ __forceinline__ float sum(float a)
	{
		if constexpr (!WIDE)
		{
			for (int o = size >> 1; o > 0; o >>= 1) a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
			return a;
		}
		else
		{
			a = warp_sum(a);
			const int warps = size >> 5;
			float* s = reinterpret_cast<float*>(slot + turn * warps);
			turn ^= 1;
			if ((lane & 31) == 0) s[lane >> 5] = a;
			asm volatile("bar.sync %0, %1;" ::"r"(1 + index), "r"(size) : "memory");
			a = (lane & 15) < warps ? s[lane & 15] : 0.0f;  // at most 16 warps: both half warps add them
#pragma unroll
			for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
			return a;
		}
	}
	// two sums over the group
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
// How a row is read: 16 bytes at a time; words of two 16-bit values, for rows that begin on any boundary (the row's whole words are then
// its elements 2 w + odd and 2 w + odd + 1, odd = 1 where the row begins in the middle of a word; the one or two values beside them are
// `edge`s of the group's first two lanes); value by value, two values that lie a group apart then make a pair.
enum { BY_QUADS = 0, BY_WORDS = 1, BY_VALUES = 2 };

// elements of an access
template <class T> __host__ __device__ constexpr int access_elems(int mode) { return mode == BY_QUADS ? 16 / (int)sizeof(T) : 2; }
// A lane's accesses to a row: `first` element of the first one; the others lie multiples of group * VEC further; a pair's second
// element lies `second` behind its first.  all(k): the access that lies k further is the row's; one(k): its first value alone is.
template <class T, int MODE>
struct RowPlace
{
	static constexpr int VEC = access_elems<T>(MODE);
	int first, n, second, edge;
	__device__ __forceinline__ RowPlace(const void* x, long long ldx, long long rows, int width, long long row, const Group& g)
	{
		const int odd = MODE == BY_WORDS ? (int)(((uintptr_t)x >> 1) + row * ldx) & 1 : 0;
		first = MODE == BY_VALUES ? g.lane : g.lane * VEC + odd;
		second = MODE == BY_VALUES ? g.size : 1;
		n = row < rows ? width : 0;
		edge = -1;
		if (MODE == BY_WORDS && n > 0)
		{
			if (g.lane == 0 && odd) edge = 0;
			if (g.lane == 1 && ((n - odd) & 1)) edge = n - 1;
		}
	}
	__device__ __forceinline__ bool all(int k) const { return first + k + (MODE == BY_QUADS ? 0 : second) < n; }
	__device__ __forceinline__ bool one(int k) const { return MODE == BY_VALUES && first + k < n && !all(k); }
	// the access that lies k further of the row that begins at `row`; what is not the row's becomes zero
	__device__ __forceinline__ void load(const T* row, int k, Pack<T, VEC>& a) const
	{
		const T* x = row + first + k;
		a.clear();
		if constexpr (MODE != BY_VALUES)
		{
			if (all(k)) a.load(x);
		}
		else
		{
			if (first + k < n) a.put(0, x[0]);
			if (all(k)) a.put(1, x[second]);
		}
	}
	__device__ __forceinline__ void store(T* row, int k, f32x2 const (&y)[VEC / 2]) const
	{
		T* x = row + first + k;
		if constexpr (MODE != BY_VALUES)
		{
			Pack<T, VEC> o;
#pragma unroll
			for (int i = 0; i < VEC / 2; ++i) o.set_pair(i, y[i]);
			if (all(k)) o.store(x);
		}
		else
		{
			float lo, hi;
			unpair2(y[0], lo, hi);
			if (first + k < n) x[0] = from_float<T>(lo);
			if (all(k)) x[second] = from_float<T>(hi);
		}
	}
	// a pair of differences without what is not the row's
	__device__ __forceinline__ f32x2 mask(f32x2 d, int k) const
	{
		if (all(k)) return d;
		if (!one(k)) return pair2(0.0f, 0.0f);
		float lo, hi;
		unpair2(d, lo, hi);
		return pair2(lo, 0.0f);
	}
	__device__ __forceinline__ T load_edge(const T* row) const { return edge >= 0 ? row[edge] : from_float<T>(0.0f); }
	// elements e and e + second of a vector of the row's columns, or `none` where there is no vector
	__device__ __forceinline__ f32x2 columns(const float* v, int e, float none) const
	{
		return pair2(v && e < n ? v[e] : none, v && e + second < n ? v[e + second] : none);
	}
};

// Groups walk the rows; a row is asked for before the row in front is worked on.  Beside HBM its instructions bound the kernel: two
// elements are worked on in one (f32x2), and gain and shift of 16-bit types stay in registers (a group only sees rows that begin on
// the same half of a word); fp32 rows have half the elements per byte, and the registers serve them better as loads under way.
//   fp32 8192 x 4096: 47 to 49 us, 5.5 to 5.7 TB/s (gain and shift in registers 54; 32 elements per lane 52)
//   bf16 8192 x 4096: 33 us; each further 8192 rows 24, of which the copy of as many bytes takes 20.5 (one value per instruction 50;
//                     32 elements per lane, gain and shift from L1, 36; a warp per row, or rows through shared memory, 43 to 50)
//   bf16 10007 x 1025: 21 us (words with a branch for the halves 31; one value at a time 42);  fp32 10007 x 1025, value by value: 37
// The registers that three CTAs per SM leave (80) do not hold 16 values of 16 bits that are not read 16 bytes at a time: 36 to 44 bytes
// a thread are spilled by words, 92 to 116 by values.  Nor do 128 hold 64 fp32 values: rows of 8193 to 16384 columns spill 236 to 492.
template <class T, int MODE, int ELEMS, bool WIDE>
__global__ void __launch_bounds__(LN_THREADS, ELEMS == 16 ? 3 : 2) norm_kernel(const LayerNormArgs p, int group)
{
	constexpr int VEC = access_elems<T>(MODE), V = ELEMS / VEC, PAIRS = VEC / 2;  // elements of an access, accesses of a lane
	__shared__ float2 slots[2 * LN_GROUP_MAX / 32];
	Group gr(group, slots);
	const int groups = blockDim.x / group;
	const long long step = (long long)gridDim.x * groups;
	const float inv_n = 1.0f / (float)p.n;
	const bool quads = MODE == BY_QUADS && (((uintptr_t)p.gain | (uintptr_t)p.shift) & 15) == 0 && p.gain && p.shift;
	typedef RowPlace<T, MODE> Place;
	constexpr bool KEEP = ELEMS == 16 && sizeof(T) == 2, EDGE = MODE == BY_WORDS;
	float gain_e = 1.0f, shift_e = 0.0f;
	T edge = from_float<T>(0.0f);
	f32x2 gain[KEEP ? V : 1][PAIRS], shift[KEEP ? V : 1][PAIRS];
	if (KEEP || EDGE)
	{
		const Place at(p.x, p.ldx, p.rows, p.n, (long long)blockIdx.x * groups + gr.index, gr);
		if (EDGE && at.edge >= 0)
		{
			if (p.gain) gain_e = p.gain[at.edge];
			if (p.shift) shift_e = p.shift[at.edge];
		}
#pragma unroll
		for (int v = 0; v < (KEEP ? V : 0); ++v)
#pragma unroll
			for (int i = 0; i < PAIRS; ++i)
			{
				const int e = at.first + v * group * VEC + 2 * i;
				gain[KEEP ? v : 0][i] = at.columns(p.gain, e, 1.0f);
				shift[KEEP ? v : 0][i] = at.columns(p.shift, e, 0.0f);
			}
	}
	auto fetch = [&](long long row, Pack<T, VEC>(&a)[V]) {
		const Place at(p.x, p.ldx, p.rows, p.n, row, gr);
		const T* x = static_cast<const T*>(p.x) + row * p.ldx;
#pragma unroll
		for (int v = 0; v < V; ++v) at.load(x, v * group * VEC, a[v]);
		if (EDGE) edge = at.load_edge(x);
	};
	long long row = (long long)blockIdx.x * groups + gr.index;
	Pack<T, VEC> next[V];
	fetch(row, next);
	// (every group of a warp walks as often as the warp's first, whose row is the smallest: the shuffles need all lanes)
	const long long walk = WIDE ? row : (long long)blockIdx.x * groups + ((int)threadIdx.x & ~31) / group;
	for (long long first = walk; first < p.rows; first += step, row += step)
	{
		const Place at(p.x, p.ldx, p.rows, p.n, row, gr);
		f32x2 x[V][PAIRS];
		f32x2 s0 = pair2(0.0f, 0.0f), s1 = s0;
#pragma unroll
		for (int v = 0; v < V; ++v)
#pragma unroll
			for (int i = 0; i < PAIRS; ++i)
			{
				x[v][i] = next[v].pair(i);
				if ((v + i) & 1) s1 = add2(s1, x[v][i]);
				else s0 = add2(s0, x[v][i]);
			}
		float a, b, xe = to_float(edge);
		fetch(row + step, next);
		unpair2(add2(s0, s1), a, b);
		if (EDGE) a += xe;
		// s / n, with the quotient's remainder: a row of equal values keeps its mean
		const float sum = gr.sum<WIDE>(a + b);
		float mean = sum * inv_n;
		if (fabsf(sum) <= 3.0e38f) mean = fmaf(fmaf(-mean, (float)p.n, sum), inv_n, mean);
		const f32x2 minus = pair2(-mean, -mean);
		s0 = s1 = pair2(0.0f, 0.0f);
#pragma unroll
		for (int v = 0; v < V; ++v)
		{
			const int k = v * group * VEC;
#pragma unroll
			for (int i = 0; i < PAIRS; ++i)
			{
				x[v][i] = add2(x[v][i], minus);
				const f32x2 d = at.mask(x[v][i], k);
				if ((v + i) & 1) s1 = fma2(d, d, s1);
				else s0 = fma2(d, d, s0);
			}
		}
		unpair2(add2(s0, s1), a, b);
		if (EDGE)
		{
			xe = at.edge >= 0 ? xe - mean : 0.0f;
			a = fmaf(xe, xe, a);
		}
		const float rstd = inverse_root(fmaf(gr.sum<WIDE>(a + b), inv_n, p.eps));
		const f32x2 scale = pair2(rstd, rstd);
		T* y = static_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
		for (int v = 0; v < V; ++v)
		{
			const int k = v * group * VEC, c = at.first + k;
			f32x2 o[PAIRS];
			if (KEEP)
			{
#pragma unroll
				for (int i = 0; i < PAIRS; ++i) o[i] = fma2(mul2(x[v][i], scale), gain[KEEP ? v : 0][i], shift[KEEP ? v : 0][i]);
			}
			else if (quads && at.all(k))
			{
#pragma unroll
				for (int i = 0; i + 1 < PAIRS; i += 2)
				{
					const float4 ga = *reinterpret_cast<const float4*>(p.gain + c + 2 * i), sh = *reinterpret_cast<const float4*>(p.shift + c + 2 * i);
					o[i] = fma2(mul2(x[v][i], scale), pair2(ga.x, ga.y), pair2(sh.x, sh.y));
					o[i + 1 < PAIRS ? i + 1 : i] = fma2(mul2(x[v][i + 1 < PAIRS ? i + 1 : i], scale), pair2(ga.z, ga.w), pair2(sh.z, sh.w));
				}
			}
			else
			{
#pragma unroll
				for (int i = 0; i < PAIRS; ++i) o[i] = fma2(mul2(x[v][i], scale), at.columns(p.gain, c + 2 * i, 1.0f), at.columns(p.shift, c + 2 * i, 0.0f));
			}
			at.store(y, k, o);
		}
		if (EDGE && at.edge >= 0) y[at.edge] = from_float<T>(fmaf(xe * rstd, gain_e, shift_e));
		if (gr.lane == 0 && at.n > 0)
		{
			if (p.mean) p.mean[row] = mean;
			if (p.rstd) p.rstd[row] = rstd;
		}
	}
}

// Rows too long for a group's registers: one CTA per row reads it three times (the second and third time from L2), 16 bytes at a time
// where every row allows it.  bf16, 800 x 40000: 44 us; value by value 69.
template <class T, int VEC>
__device__ __forceinline__ void load_values(const T* p, float (&f)[VEC])
{
	if constexpr (VEC == 1) f[0] = to_float(p[0]);
	else
	{
		Pack<T, VEC> a;
		a.load(p);
#pragma unroll
		for (int i = 0; i < VEC / 2; ++i) unpair2(a.pair(i), f[2 * i], f[2 * i + 1]);
	}
}
// VEC values of a vector of the columns, or `none` where there is no vector
template <int VEC>
__device__ __forceinline__ void load_columns(const float* p, long long c, float none, float (&f)[VEC])
{
	if constexpr (VEC == 1) f[0] = p ? p[c] : none;
	else
	{
#pragma unroll
		for (int i = 0; i < VEC; i += 4)
		{
			const float4 v = p ? *reinterpret_cast<const float4*>(p + c + i) : make_float4(none, none, none, none);
			f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
		}
	}
}
template <class T, int VEC>
__device__ __forceinline__ void store_values(T* p, const float (&f)[VEC])
{
	if constexpr (VEC == 1) p[0] = from_float<T>(f[0]);
	else
	{
		Pack<T, VEC> a;
#pragma unroll
		for (int i = 0; i < VEC / 2; ++i) a.set_pair(i, pair2(f[2 * i], f[2 * i + 1]));
		a.store(p);
	}
}
template <class T, int VEC>
__global__ void __launch_bounds__(LN_GROUP_MAX) norm_long_kernel(const LayerNormArgs p)
{
	__shared__ float2 slots[2 * LN_GROUP_MAX / 32];
	Group gr(LN_GROUP_MAX, slots);
	const float inv_n = 1.0f / (float)p.n;
	const int from = threadIdx.x * VEC, step = LN_GROUP_MAX * VEC;
	for (long long row = blockIdx.x; row < p.rows; row += gridDim.x)
	{
		const T* x = static_cast<const T*>(p.x) + row * p.ldx;
		T* y = static_cast<T*>(p.y) + row * p.ldy;
		float s = 0.0f, f[VEC];
#pragma unroll 4
		for (long long c = from; c < p.n; c += step)
		{
			load_values<T, VEC>(x + c, f);
#pragma unroll
			for (int i = 0; i < VEC; ++i) s += f[i];
		}
		const float mean = gr.sum<true>(s) / (float)p.n;
		float q = 0.0f;
#pragma unroll 4
		for (long long c = from; c < p.n; c += step)
		{
			load_values<T, VEC>(x + c, f);
#pragma unroll
			for (int i = 0; i < VEC; ++i) q = fmaf(f[i] - mean, f[i] - mean, q);
		}
		const float rstd = 1.0f / sqrtf(gr.sum<true>(q) * inv_n + p.eps);
#pragma unroll 4
		for (long long c = from; c < p.n; c += step)
		{
			float gain[VEC], shift[VEC];
			load_values<T, VEC>(x + c, f);
			load_columns<VEC>(p.gain, c, 1.0f, gain);
			load_columns<VEC>(p.shift, c, 0.0f, shift);
#pragma unroll
			for (int i = 0; i < VEC; ++i) f[i] = fmaf((f[i] - mean) * rstd, gain[i], shift[i]);
			store_values<T, VEC>(y + c, f);
		}
		if (threadIdx.x == 0)
		{
			if (p.mean) p.mean[row] = mean;
			if (p.rstd) p.rstd[row] = rstd;
		}
	}
}

// ---- backward ------------------------------------------------------------------------------------------------
// The same groups; both row sums in one exchange.  A lane keeps the same columns for all its rows and adds their dgain and dshift up in
// registers; a CTA's groups are added in a fixed order and leave as one partial row, which norm_columns_kernel adds up: no atomics, two
// runs give the same bits.  Every difference is scaled as it is taken, xh = (x - mu) r: sums of g (x - mu) and powers of r beside
// them would leave fp32's range where activations are very large or very small.
//   bf16 10007 x 1025: 35 us (one value at a time 164);  fp32 10007 x 1025, value by value: 84;  bf16 30000 x 100: 19
// A row's values, their columns' sums and the next row are more than the 128 registers of 512 threads: every instantiation of
// norm_backward_kernel spills 128 to 344 bytes a thread.
// A CTA's sums of the columns: its groups' are added in a fixed order in `sums`, [groups or (in-warp groups) warps][n], and leave as
// one partial row.  A lane's access v begins at column first + v * group * VEC.
template <bool APART, bool WIDE, int V, int PAIRS>
__device__ __forceinline__ void leave_columns(const LayerNormArgs& p, const Group& gr, int first, f32x2 (&dg)[V][PAIRS], f32x2 (&ds)[V][PAIRS], int edge, float2 dedge, float2* sums)
{
	const int group = gr.size, second = APART ? group : 1;
	if (!WIDE)
	{
		// the warp's groups hold the same columns on lanes that are a group apart
#pragma unroll
		for (int v = 0; v < V; ++v)
#pragma unroll
			for (int i = 0; i < PAIRS; ++i)
				for (int o = group; o < 32; o <<= 1)
				{
					dg[v][i] = add2(dg[v][i], __shfl_xor_sync(0xFFFFFFFFu, dg[v][i], o));
					ds[v][i] = add2(ds[v][i], __shfl_xor_sync(0xFFFFFFFFu, ds[v][i], o));
				}
		for (int o = group; o < 32; o <<= 1)
		{
			dedge.x += __shfl_xor_sync(0xFFFFFFFFu, dedge.x, o);
			dedge.y += __shfl_xor_sync(0xFFFFFFFFu, dedge.y, o);
		}
	}
	const int parts = WIDE ? (int)blockDim.x / group : (int)blockDim.x / 32;
	const int part = WIDE ? gr.index : (int)threadIdx.x / 32;
	float2* out = parts == 1 ? p.part + (long long)blockIdx.x * p.n : sums + (long long)part * p.n;
	if (WIDE || (int)(threadIdx.x & 31) < group)
	{
#pragma unroll
		for (int v = 0; v < V; ++v)
#pragma unroll
			for (int i = 0; i < PAIRS; ++i)
			{
				const int e = first + v * group * 2 * PAIRS + 2 * i, f = e + second;
				float g0, g1, s0, s1;
				unpair2(dg[v][i], g0, g1);
				unpair2(ds[v][i], s0, s1);
				if ((APART ? e : f) < p.n) out[e] = make_float2(g0, s0);
				if (f < p.n) out[f] = make_float2(g1, s1);
			}
		if (edge >= 0) out[edge] = dedge;
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

template <class T, int MODE, bool WIDE>
__global__ void __launch_bounds__(LN_GROUP_MAX, 1) norm_backward_kernel(const LayerNormArgs p, int group)
{
	constexpr int VEC = access_elems<T>(MODE), V = LN_ELEMS / VEC, PAIRS = VEC / 2;
	extern __shared__ float2 sums[];  // [groups or (in-warp groups) warps][n]
	__shared__ float2 slots[2 * LN_GROUP_MAX / 32];
	Group gr(group, slots);
	const int groups = blockDim.x / group;
	const long long step = (long long)gridDim.x * groups;
	typedef RowPlace<T, MODE> Place;
	const float inv_n = 1.0f / (float)p.n;
	const f32x2 zero = pair2(0.0f, 0.0f);
	cudaTriggerProgrammaticLaunchCompletion();
	f32x2 gain[V][PAIRS], dg[V][PAIRS], ds[V][PAIRS];
	long long row = (long long)blockIdx.x * groups + gr.index;
	const Place column(p.x, p.ldx, row + 1, p.n, row, gr);  // (of a group without rows too: it leaves zeros)
#pragma unroll
	for (int v = 0; v < V; ++v)
#pragma unroll
		for (int i = 0; i < PAIRS; ++i)
		{
			gain[v][i] = column.columns(p.gain, column.first + v * group * VEC + 2 * i, 1.0f);
			dg[v][i] = ds[v][i] = zero;
		}
	constexpr bool EDGE = MODE == BY_WORDS;
	const float gain_e = EDGE && p.gain && column.edge >= 0 ? p.gain[column.edge] : 1.0f;
	float dg_e = 0.0f, ds_e = 0.0f;
	T xe_n = from_float<T>(0.0f), de_n = xe_n;
	Pack<T, VEC> xn[V], dn[V];
	float mean_n = 0.0f, rstd_n = 0.0f;
	auto fetch = [&](long long row) {
		const Place at(p.x, p.ldx, p.rows, p.n, row, gr);
		if (row < p.rows)
		{
			mean_n = p.mean[row];
			rstd_n = p.rstd[row];
		}
		const T *x = static_cast<const T*>(p.x) + row * p.ldx, *dy = static_cast<const T*>(p.dy) + row * p.lddy;
#pragma unroll
		for (int v = 0; v < V; ++v)
		{
			at.load(x, v * group * VEC, xn[v]);
			at.load(dy, v * group * VEC, dn[v]);
		}
		if (EDGE)
		{
			xe_n = at.load_edge(x);
			de_n = at.load_edge(dy);
		}
	};
	fetch(row);
	const long long walk = WIDE ? row : (long long)blockIdx.x * groups + ((int)threadIdx.x & ~31) / group;
	for (long long first = walk; first < p.rows; first += step, row += step)
	{
		const Place at(p.x, p.ldx, p.rows, p.n, row, gr);
		const f32x2 minus = pair2(-mean_n, -mean_n), scale = pair2(rstd_n, rstd_n);
		const float rstd = rstd_n;
		f32x2 xh[V][PAIRS], g[V][PAIRS];
		f32x2 a2 = zero, b2 = zero;
#pragma unroll
		for (int v = 0; v < V; ++v)
#pragma unroll
			for (int i = 0; i < PAIRS; ++i)
			{
				// (what is not the row's has a dy of zero, and a difference that means nothing)
				const f32x2 dy = dn[v].pair(i);
				xh[v][i] = mul2(at.mask(add2(xn[v].pair(i), minus), v * group * VEC), scale);
				g[v][i] = mul2(dy, gain[v][i]);
				a2 = add2(a2, g[v][i]);
				b2 = fma2(g[v][i], xh[v][i], b2);
				dg[v][i] = fma2(dy, xh[v][i], dg[v][i]);
				ds[v][i] = add2(ds[v][i], dy);
			}
		float a, b, c, e, xhe = 0.0f, ge = 0.0f;
		unpair2(a2, a, c);
		unpair2(b2, b, e);
		if (EDGE && at.edge >= 0)
		{
			const float dy = to_float(de_n);
			xhe = (to_float(xe_n) - mean_n) * rstd;
			ge = dy * gain_e;
			a += ge;
			b = fmaf(ge, xhe, b);
			dg_e = fmaf(dy, xhe, dg_e);
			ds_e += dy;
		}
		fetch(row + step);
		if (!p.dx) continue;
		const float2 s = gr.sum<WIDE>(a + c, b + e);
		if (at.n == 0) continue;
		const float ma = -s.x * inv_n * rstd, mb = -s.y * inv_n * rstd;
		const f32x2 ma2 = pair2(ma, ma), mb2 = pair2(mb, mb);
		T* dx = static_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
		for (int v = 0; v < V; ++v)
		{
			f32x2 o[PAIRS];
#pragma unroll
			for (int i = 0; i < PAIRS; ++i) o[i] = fma2(g[v][i], scale, fma2(xh[v][i], mb2, ma2));
			at.store(dx, v * group * VEC, o);
		}
		if (EDGE && at.edge >= 0) dx[at.edge] = from_float<T>(fmaf(ge, rstd, fmaf(xhe, mb, ma)));
	}
	if (p.part) leave_columns<MODE == BY_VALUES, WIDE>(p, gr, column.first, dg, ds, column.edge, make_float2(dg_e, ds_e), sums);
}

// Rows that 16-byte accesses can read: they are copied to shared memory several rows ahead, each lane its own accesses, and read
// there twice, so that a lane's registers hold only what outlives a row.  One CTA of 512 threads per SM: 768, with 80 registers each, spill.
//   fp32 8192 x 4096: 72 us, 5.6 TB/s (one row ahead in registers 110);  bf16: 50 us, each further 8192 rows 31: as the copy of as
//   many bytes.  What is above that is the start, the CTAs' sums and the columns' kernel.
template <class T> __host__ __device__ constexpr int quads_stages() { return 208 * 1024 / (LN_GROUP_MAX * 2 * LN_ELEMS * (int)sizeof(T)); }
template <class T> constexpr size_t quads_bytes(int threads) { return (size_t)threads * 2 * LN_ELEMS * sizeof(T) * quads_stages<T>(); }
// the columns' sums of a CTA's groups, or of the warps that hold several: at most 16 rows of 512 columns, or as many values in fewer, longer
// rows; rows of words have a column more
constexpr size_t sums_bytes = (size_t)(LN_GROUP_MAX * LN_ELEMS + LN_GROUP_MAX / 32) * sizeof(float2);
template <class T, bool WIDE>
__global__ void __launch_bounds__(LN_GROUP_MAX, 1) norm_backward_quads_kernel(const LayerNormArgs p, int group)
{
	constexpr int VEC = access_elems<T>(BY_QUADS), V = LN_ELEMS / VEC, PAIRS = VEC / 2, STAGES = quads_stages<T>();
	extern __shared__ uint4 ahead[];  // [STAGES][x, dy][V][threads]; at the end the columns' sums
	__shared__ float2 slots[2 * LN_GROUP_MAX / 32];
	Group gr(group, slots);
	const int groups = blockDim.x / group;
	const long long step = (long long)gridDim.x * groups;
	const float inv_n = 1.0f / (float)p.n;
	const f32x2 zero = pair2(0.0f, 0.0f);
	cudaTriggerProgrammaticLaunchCompletion();
	const int first_c = gr.lane * VEC, hop = group * VEC;
	uint4* const mine = ahead + threadIdx.x;
	f32x2 gain[V][PAIRS], dg[V][PAIRS], ds[V][PAIRS];
#pragma unroll
	for (int v = 0; v < V; ++v)
#pragma unroll
		for (int i = 0; i < PAIRS; ++i)
		{
			const int e = first_c + v * hop + 2 * i;
			gain[v][i] = p.gain && e < p.n ? pair2(p.gain[e], p.gain[e + 1]) : pair2(1.0f, 1.0f);
			dg[v][i] = ds[v][i] = zero;
		}
	float mean_n = 0.0f, rstd_n = 0.0f;
	auto fetch = [&](long long row, int stage) {
		const bool is = row < p.rows;
		const T *x = static_cast<const T*>(p.x) + (is ? row * p.ldx : 0), *dy = static_cast<const T*>(p.dy) + (is ? row * p.lddy : 0);
#pragma unroll
		for (int v = 0; v < V; ++v)
		{
			const int c = first_c + v * hop;
			const bool in = is && c < p.n;
			copy_ahead(mine + (2 * stage * V + v) * (int)blockDim.x, x + (in ? c : 0), in);
			copy_ahead(mine + ((2 * stage + 1) * V + v) * (int)blockDim.x, dy + (in ? c : 0), in);
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
	};
	auto fetch_statistics = [&](long long row) {
		if (row >= p.rows) return;
		mean_n = p.mean[row];
		rstd_n = p.rstd[row];
	};
	long long row = (long long)blockIdx.x * groups + gr.index;
	for (int i = 0; i < STAGES; ++i) fetch(row + i * step, i);
	fetch_statistics(row);
	int stage = 0;
	const long long walk = WIDE ? row : (long long)blockIdx.x * groups + ((int)threadIdx.x & ~31) / group;
	for (long long first = walk; first < p.rows; first += step, row += step)
	{
		const f32x2 minus = pair2(-mean_n, -mean_n), scale = pair2(rstd_n, rstd_n);
		const float rstd = rstd_n;
		f32x2 a2 = zero, b2 = zero;
		asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
		fetch_statistics(row + step);
		const uint4 *xs = mine + 2 * stage * V * (int)blockDim.x, *dys = xs + V * (int)blockDim.x;
#pragma unroll
		for (int v = 0; v < V; ++v)
		{
			Pack<T, VEC> xv, dv;  // (what is not the row's has a dy of zero, and a difference that means nothing)
			xv.set(xs[v * (int)blockDim.x]);
			dv.set(dys[v * (int)blockDim.x]);
#pragma unroll
			for (int i = 0; i < PAIRS; ++i)
			{
				const f32x2 dy = dv.pair(i), xh = mul2(add2(xv.pair(i), minus), scale), g = mul2(dy, gain[v][i]);
				a2 = add2(a2, g);
				b2 = fma2(g, xh, b2);
				dg[v][i] = fma2(dy, xh, dg[v][i]);
				ds[v][i] = add2(ds[v][i], dy);
			}
		}
		if (p.dx)
		{
			float a, b, c, e;
			unpair2(a2, a, c);
			unpair2(b2, b, e);
			const float2 s = gr.sum<WIDE>(a + c, b + e);
			const float ma = -s.x * inv_n, mb = -s.y * inv_n * rstd;
			const f32x2 ma2 = pair2(ma, ma), mb2 = pair2(mb, mb);
			T* dx = static_cast<T*>(p.dx) + row * p.lddx + first_c;
			if (row < p.rows)
			{
#pragma unroll
				for (int v = 0; v < V; ++v)
				{
					Pack<T, VEC> xv, dv, o;
					xv.set(xs[v * (int)blockDim.x]);
					dv.set(dys[v * (int)blockDim.x]);
#pragma unroll
					for (int i = 0; i < PAIRS; ++i)
						o.set_pair(i, mul2(fma2(dv.pair(i), gain[v][i], fma2(add2(xv.pair(i), minus), mb2, ma2)), scale));
					if (first_c + v * hop < p.n) o.store(dx + v * hop);
				}
			}
		}
		fetch(row + STAGES * step, stage);
		stage = stage + 1 == STAGES ? 0 : stage + 1;
	}
	asm volatile("cp.async.wait_all;" ::: "memory");
	__syncthreads();
	if (p.part) leave_columns<false, WIDE>(p, gr, first_c, dg, ds, -1, make_float2(0.0f, 0.0f), reinterpret_cast<float2*>(ahead));
}

// Long rows: dx by a CTA per row in two passes ...
template <class T, int VEC>
__global__ void __launch_bounds__(LN_GROUP_MAX) norm_backward_long_kernel(const LayerNormArgs p)
{
	__shared__ float2 slots[2 * LN_GROUP_MAX / 32];
	Group gr(LN_GROUP_MAX, slots);
	const float inv_n = 1.0f / (float)p.n;
	const int from = threadIdx.x * VEC, step = LN_GROUP_MAX * VEC;
	for (long long row = blockIdx.x; row < p.rows; row += gridDim.x)
	{
		const T* x = static_cast<const T*>(p.x) + row * p.ldx;
		const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
		T* dx = static_cast<T*>(p.dx) + row * p.lddx;
		const float mean = p.mean[row], rstd = p.rstd[row];
		float a = 0.0f, b = 0.0f, f[VEC], d[VEC], gain[VEC];
#pragma unroll 2
		for (long long c = from; c < p.n; c += step)
		{
			load_values<T, VEC>(x + c, f);
			load_values<T, VEC>(dy + c, d);
			load_columns<VEC>(p.gain, c, 1.0f, gain);
#pragma unroll
			for (int i = 0; i < VEC; ++i)
			{
				const float g = d[i] * gain[i];
				a += g;
				b = fmaf(g, (f[i] - mean) * rstd, b);
			}
		}
		const float2 s = gr.sum<true>(a, b);
		const float ma = s.x * inv_n, mb = s.y * inv_n;
#pragma unroll 2
		for (long long c = from; c < p.n; c += step)
		{
			load_values<T, VEC>(x + c, f);
			load_values<T, VEC>(dy + c, d);
			load_columns<VEC>(p.gain, c, 1.0f, gain);
#pragma unroll
			for (int i = 0; i < VEC; ++i) f[i] = rstd * (fmaf(d[i], gain[i], -ma) - (f[i] - mean) * rstd * mb);
			store_values<T, VEC>(dx + c, f);
		}
	}
}
// ... and the columns' sums over a slice of the rows
template <class T, int VEC>
__global__ void __launch_bounds__(LN_THREADS) norm_slices_kernel(const LayerNormArgs p, int slices)
{
	const long long c = ((long long)blockIdx.x * LN_THREADS + threadIdx.x) * VEC;
	if (c >= p.n) return;
	const T* x = static_cast<const T*>(p.x) + c;
	const T* dy = static_cast<const T*>(p.dy) + c;
	float2 t[VEC];
#pragma unroll
	for (int i = 0; i < VEC; ++i) t[i] = make_float2(0.0f, 0.0f);
#pragma unroll 4
	for (long long row = blockIdx.y; row < p.rows; row += slices)
	{
		float f[VEC], d[VEC];
		load_values<T, VEC>(x + row * p.ldx, f);
		load_values<T, VEC>(dy + row * p.lddy, d);
		const float mean = p.mean[row], rstd = p.rstd[row];
#pragma unroll
		for (int i = 0; i < VEC; ++i)
		{
			t[i].x = fmaf(d[i], (f[i] - mean) * rstd, t[i].x);
			t[i].y += d[i];
		}
	}
#pragma unroll
	for (int i = 0; i < VEC; ++i)
		if (VEC == 1) p.part[(long long)blockIdx.y * p.n + c] = t[i];
		else if (i % 2 == 0) reinterpret_cast<float4*>(p.part + (long long)blockIdx.y * p.n + c)[i / 2] = make_float4(t[i].x, t[i].y, t[i + 1 < VEC ? i + 1 : i].x, t[i + 1 < VEC ? i + 1 : i].y);
}

// dgain | dshift from `parts` partial rows: 32 columns per CTA, LN_SLICES slices of the partials, added in a fixed order
__global__ void __launch_bounds__(32 * LN_SLICES) norm_columns_kernel(const float2* part, int parts, int n, float* dgain, float* dshift)
{
	__shared__ float2 sums[LN_SLICES][33];
	const int k = threadIdx.x & 31, slice = threadIdx.x >> 5;
	const long long c = (long long)blockIdx.x * 32 + k;
	cudaGridDependencySynchronize();
	float2 t = make_float2(0.0f, 0.0f);
	if (c < n)
	{
#pragma unroll 5
		for (int r = slice; r < parts; r += LN_SLICES)
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
	for (int s = 1; s < LN_SLICES; ++s)
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

// Do all rows of all tensors consist of whole pieces of so many bytes?
bool aligned(const LayerNormArgs& a, int size, int bytes)
{
	auto ok = [&](const void* p, long long ld) { return !p || ((uintptr_t)p % bytes == 0 && (ld * size) % bytes == 0); };
	return ((long long)a.n * size) % bytes == 0 && ok(a.x, a.ldx) && ok(a.y, a.ldy) && ok(a.dy, a.lddy) && ok(a.dx, a.lddx);
}

// and the same of the vectors of columns, which long rows read 16 bytes at a time
bool columns_aligned(const LayerNormArgs& a) { return (((uintptr_t)a.gain | (uintptr_t)a.shift) & 15) == 0; }

// Threads and CTAs of the backward kernel, each CTA of which leaves one partial row: one CTA per SM, with two or more groups where
// a row is short enough; but smaller ones where there would be fewer than SMs (1024 x 256 in fp32 runs on 128 SMs, not on 32).
void backward_shape(long long rows, int group, int* threads, int* ctas)
{
	int t = LN_GROUP_MAX;
	while (t > 64 && t / 2 >= group && (rows + t / group - 1) / (t / group) < LN_SMS) t /= 2;
	*threads = group <= t ? group * (t / group) : group;
	const int groups = *threads / group;
	*ctas = (int)std::min<long long>(LN_SMS, (rows + groups - 1) / groups);
}
bool backward_long(int n) { return n > LN_GROUP_MAX * LN_ELEMS; }
// Lanes of a row of whole words and their edges, which take two.
int mode_lanes(int n, int elems, int mode) { return mode == BY_WORDS ? std::max(2, group_lanes(n / 2 * 2, elems)) : group_lanes(n, elems); }
int backward_slices(long long rows) { return (int)(rows < 32 ? rows : 32); }

template <class T, int MODE, int ELEMS>
cudaError_t forward_elems(const LayerNormArgs& a, cudaStream_t s)
{
	const int group = mode_lanes(a.n, ELEMS, MODE);
	const int threads = group_threads(group);
	const int groups = threads / group;
	const long long want = (a.rows + groups - 1) / groups;
	// (LN_SMS is even: a group that walks sees rows of one kind only, where every other row begins in the middle of a word)
	const long long most = (long long)LN_SMS * std::max(1, (ELEMS == 16 ? 768 : 512) / threads);
	const unsigned grid = (unsigned)(want < most ? want : most);
	// (more than 16 elements per lane are rows of more than 4096: more lanes than a warp's)
	if constexpr (ELEMS == 16)
		if (group <= 32)
		{
			norm_kernel<T, MODE, ELEMS, false><<<grid, threads, 0, s>>>(a, group);
			return cudaGetLastError();
		}
	norm_kernel<T, MODE, ELEMS, true><<<grid, threads, 0, s>>>(a, group);
	return cudaGetLastError();
}

template <class T, int MODE>
cudaError_t forward_mode(const LayerNormArgs& a, cudaStream_t s)
{
	if (a.n <= LN_THREADS * 16) return forward_elems<T, MODE, 16>(a, s);
	return a.n <= LN_THREADS * 32 ? forward_elems<T, MODE, 32>(a, s) : forward_elems<T, MODE, 64>(a, s);
}

template <class T, int MODE>
cudaError_t backward_mode(const LayerNormArgs& a, int* ctas, cudaStream_t s)
{
	const int group = mode_lanes(a.n, LN_ELEMS, MODE);
	int threads, grid;
	backward_shape(a.rows, group, &threads, &grid);
	*ctas = grid;
	const int parts = group > 32 ? threads / group : threads / 32;
	size_t smem = parts > 1 ? (size_t)parts * a.n * sizeof(float2) : 0;
	constexpr size_t most = MODE == BY_QUADS ? quads_bytes<T>(LN_GROUP_MAX) : sums_bytes;
	auto go = [&](void (*kernel)(LayerNormArgs, int)) {
		int sms = 0;
		if (smem > most) return cudaErrorInvalidValue;
		if (cudaError_t e = prepare_tc_launch(reinterpret_cast<const void*>(kernel), (int)most, &sms)) return e;
		kernel<<<grid, threads, smem, s>>>(a, group);
		return cudaGetLastError();
	};
	if constexpr (MODE == BY_QUADS)
	{
		smem = std::max(smem, quads_bytes<T>(threads));
		return group > 32 ? go(norm_backward_quads_kernel<T, true>) : go(norm_backward_quads_kernel<T, false>);
	}
	else return group > 32 ? go(norm_backward_kernel<T, MODE, true>) : go(norm_backward_kernel<T, MODE, false>);
}

// Two tensors whose rows begin on the same half of a word.
bool alike(const void* x, long long ldx, const void* y, long long ldy) { return (((uintptr_t)x ^ (uintptr_t)y) & 2) == 0 && ((ldx ^ ldy) & 1) == 0; }

template <class T>
cudaError_t forward_type(const LayerNormArgs& a, cudaStream_t s)
{
	if (a.n > LN_THREADS * 64)
	{
		const unsigned grid = (unsigned)std::min<long long>(a.rows, LN_SMS * 4);
		if (aligned(a, sizeof(T), 16) && columns_aligned(a)) norm_long_kernel<T, 16 / sizeof(T)><<<grid, LN_GROUP_MAX, 0, s>>>(a);
		else norm_long_kernel<T, 1><<<grid, LN_GROUP_MAX, 0, s>>>(a);
		return cudaGetLastError();
	}
	if (aligned(a, sizeof(T), 16)) return forward_mode<T, BY_QUADS>(a, s);
	if constexpr (sizeof(T) == 2)
		if (alike(a.x, a.ldx, a.y, a.ldy)) return forward_mode<T, BY_WORDS>(a, s);
	return forward_mode<T, BY_VALUES>(a, s);
}

template <class T, int VEC>
cudaError_t backward_long_rows(const LayerNormArgs& a, int parts, cudaStream_t s)
{
	if (a.part) norm_slices_kernel<T, VEC><<<dim3((unsigned)((a.n + LN_THREADS * VEC - 1) / (LN_THREADS * VEC)), (unsigned)parts), LN_THREADS, 0, s>>>(a, parts);
	if (cudaError_t e = cudaGetLastError()) return e;
	if (a.dx) norm_backward_long_kernel<T, VEC><<<(unsigned)std::min<long long>(a.rows, LN_SMS * 4), LN_GROUP_MAX, 0, s>>>(a);
	return cudaGetLastError();
}

template <class T>
cudaError_t backward_type(const LayerNormArgs& a, cudaStream_t s)
{
	int parts;
	if (backward_long(a.n))
	{
		parts = backward_slices(a.rows);
		const cudaError_t e = aligned(a, sizeof(T), 16) && columns_aligned(a) ? backward_long_rows<T, 16 / sizeof(T)>(a, parts, s) : backward_long_rows<T, 1>(a, parts, s);
		if (e != cudaSuccess) return e;
	}
	else
	{
		cudaError_t e = cudaErrorInvalidValue;
		// by words: in a warp of several groups the columns' sums must lie on the same lanes of each
		const bool words = sizeof(T) == 2 && (mode_lanes(a.n, LN_ELEMS, BY_WORDS) > 32 || (a.ldx & 1) == 0) && alike(a.x, a.ldx, a.dy, a.lddy) &&
		                   (!a.dx || alike(a.x, a.ldx, a.dx, a.lddx));
		if (aligned(a, sizeof(T), 16)) e = backward_mode<T, BY_QUADS>(a, &parts, s);
		else if (!words) e = backward_mode<T, BY_VALUES>(a, &parts, s);
		else if constexpr (sizeof(T) == 2) e = backward_mode<T, BY_WORDS>(a, &parts, s);
		if (e != cudaSuccess) return e;
	}
	if (!a.part) return cudaSuccess;
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned)((a.n + 31) / 32));
	cfg.blockDim = dim3(32 * LN_SLICES);
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
	if (backward_long(n)) return (size_t)backward_slices(rows);
	return (size_t)std::min<long long>(rows, LN_SMS);
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
