// Orthogonalisation of small matrices: one CTA per matrix, everything in its shared memory (the mathematics: orthogonalize.cu).
// The same program on the same tensor-core operands, but no copies, no grid barriers and no symmetry: what bounds
// a round here is the chain MMAs -> commit -> tensor-memory loads -> parts into shared memory -> block barrier, 1.5
// us against 6 of the cooperative kernel (its barrier alone takes one).
//
// Layout: a matrix of parts is stored in chunks of 64 columns, [chunk][hi | lo][row][64 halfs], rows of 128 bytes in the 128-byte
// swizzle, `rows` = the short side rounded up to 16, filled with zeros.  The same bytes are a K-major operand (rows by k = columns,
// for X X^T and the products of symmetric matrices) and an MN-major one (k = rows by columns, for R X), and hi and lo as
// they follow one another are one operand of twice the size: K-major twice the rows, MN-major twice the columns.  An MMA
// always takes 128 rows of its first operand; those behind the matrix's are whatever lies there and only reach rows of the
// accumulator that nobody reads.
// X <- q X + Q X and R <- b A + c A^2 are written over what they are made of: the MMAs that read a chunk are done when it is written,
// and every element's own old value is read by the thread that writes it.
#include <string.h>

#include <algorithm>

#include "ortho_device.cuh"

namespace glb {
namespace {

constexpr int SM_WARPS = 16;                        // epilogue warps: four for each quarter of tensor memory's lanes
constexpr int SM_THREADS = 32 * (SM_WARPS + 1);     // and one that multiplies
// 16-k steps of a square product that an accumulator takes before it is drained: sums of squares lose half a unit in the last place with
// every addition.  Random 64 x 512 against 64 bits, relative to the error of fp32 products: 8 steps 2.0, 4 steps 1.9, two 1.2, one 0.8;
// 112 x 300 takes 101, 107, 130 and 179 us.
constexpr int SM_K = 2;
constexpr int SM_TMEM = 512, SM_BUFFER = 256;       // columns: all, and of one of the two accumulators
constexpr int SM_SMEM = 227 * 1024;

struct SmMat
{
	OrthoMatrix m;
	int p, q, tall, vector;
	int rows, chunks;  // rows of a chunk, chunks of X
};
struct SmParams
{
	OrProgram prog;
	SmMat mat[ORTHO_MAX_MATRICES];
	float coef[ORTHO_MAX_STEPS][3];
	int count, steps, type, step, nesterov, reset;
	float mu, decay, eps, s0;
	int* status;
	int* bad;
};

__host__ __device__ inline int small_part(int rows) { return rows * 128; }  // bytes of hi (or lo) of a chunk

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8])
{
	asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
	             : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
	             : "r"(taddr));
}

// A single row or column: X stays U times a number, A = X X^T is a number, and so are the steps: they are done in double, and the result
// is rounded once (three fp16 products: 1 to 2e-6 off, since every step multiplies the one number's rounding).
__device__ __noinline__ void orthogonalize_vector(const SmParams& P, const SmMat& M, double* warp_sums)
{
	const OrthoMatrix& m = M.m;
	auto at = [&](int e, long long ld) { return m.cols == 1 ? e * ld : (long long)e; };
	double sum = 0.0;
#pragma unroll 4
	for (int e = threadIdx.x; e < M.q; e += SM_THREADS)
	{
		float u = load_typed(m.grad, at(e, m.ld_grad), P.type);
		if (P.step)
		{
			const float v = fmaf(P.mu, m.mom[at(e, m.ld_mom)], u);
			m.mom_out[at(e, m.ld_mom)] = v;
			u = P.nesterov ? fmaf(P.mu, v, u) : v;
		}
		sum = fma((double)u, (double)u, sum);
	}
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
	if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x / 32] = sum;
	__syncthreads();
	sum = 0.0;
	for (int w = 0; w < SM_THREADS / 32; ++w) sum += warp_sums[w];
	const double inv = inverse_norm(sum, P.eps);
	double a = sum * inv * inv, factor = inv;
	for (int k = 0; k < P.steps; ++k)
	{
		const double f = (double)P.coef[k][0] + a * ((double)P.coef[k][1] + a * (double)P.coef[k][2]);
		factor *= f;
		a *= f * f;
	}
	const float keep = 1.0f - m.lr * P.decay;
	bool finite = true;
#pragma unroll 4
	for (int e = threadIdx.x; e < M.q; e += SM_THREADS)
	{
		float u;
		if (P.step)
		{
			u = m.mom_out[at(e, m.ld_mom)];
			if (P.nesterov) u = fmaf(P.mu, u, load_typed(m.grad, at(e, m.ld_grad), P.type));
		}
		else u = load_typed(m.grad, at(e, m.ld_grad), P.type);
		const float o = (float)(u * factor);
		if (!P.step)
		{
			store_typed(m.out, at(e, m.ld_out), o, P.type);
			continue;
		}
		const float w = fmaf(-m.lr, o, keep * m.w[at(e, m.ld_w)]);
		finite = finite && isfinite(w);
		m.w_out[at(e, m.ld_w)] = w;
	}
	if (P.step && P.bad && !finite) atomicOr(P.bad, 1);
}

__global__ void __launch_bounds__(SM_THREADS, 1) ortho_small_kernel(const __grid_constant__ SmParams P)
{
	extern __shared__ uint8_t smem_raw[];
	__shared__ uint64_t bars[5];  // full[2], empty[2], given up
	__shared__ uint32_t tmem_slot;
	__shared__ int aborted;
	__shared__ double warp_sums[SM_WARPS + 1];
	__shared__ OrOp ops[OR_MAX_OPS];  // (from constant memory every operation would cost a miss on the way)
	const SmMat& M = P.mat[blockIdx.x];
	const OrthoMatrix& m = M.m;
	if (M.vector)
	{
		if (blockIdx.x == 0 && threadIdx.x == 0 && P.reset) *P.status = 0;
		orthogonalize_vector(P, M, warp_sums);
		cudaGridDependencySynchronize();  // (it may have been let in beside the kernel in front, which the stream's next work waits for too)
		return;
	}
	const int count = P.prog.count;
	for (int i = threadIdx.x; i < count; i += SM_THREADS) ops[i] = P.prog.op[i];
	const uint32_t raw = smem_u32(smem_raw);
	const uint32_t base = (raw + 1023u) & ~1023u;
	uint8_t* gen = smem_raw + (base - raw);
	const uint32_t bar0 = smem_u32(bars);
	volatile int* abort_flag = &aborted;
	const int warp = __shfl_sync(0xFFFFFFFFu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
	const int rows = M.rows, part = small_part(rows), chunk = 2 * part;
	const uint32_t xbase = base + (uint32_t)((rows + 63) / 64 * chunk);
	auto at = [&](int id) -> uint32_t { return id >= ID_X ? xbase : base; };  // where a matrix of parts begins: there is one X, and A and R are one

	if (threadIdx.x == 0)
	{
		for (int b = 0; b < 2; ++b)
		{
			mbar_init(bar0 + 8 * b, 1);
			mbar_init(bar0 + 16 + 8 * b, SM_WARPS);
		}
		mbar_init(bar0 + 32, 1);
		aborted = 0;
		asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
		if (blockIdx.x == 0 && P.reset) *P.status = 0;
	}
	if (warp == SM_WARPS)
	{
		asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(SM_TMEM) : "memory");
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
	}

	// ---- sum of squares (in double: a product of two floats is exact there and does not leave its range), X filled with zeros.
	// Four neighbours of a row per thread and turn, four turns' loads ahead of their use; the first four turns stay in registers.
	const unsigned quads = ((unsigned)m.cols + 3) / 4, total = (unsigned)m.rows * quads;
	const bool wg = (((uintptr_t)m.grad | (uintptr_t)(m.ld_grad * (P.type == GL_F32 ? 4 : 2))) & (P.type == GL_F32 ? 15 : 7)) == 0;
	const bool wm = P.step && (((uintptr_t)m.mom | (uintptr_t)m.mom_out | (uintptr_t)(m.ld_mom * 4)) & 15) == 0;
	auto fetch = [&](unsigned e, bool again, float (&w)[4], float (&v)[4], long long& i, int& left, unsigned& r, unsigned& c) {
		r = e / quads;
		c = (e - r * quads) * 4;
		left = e < total ? m.cols - (int)c : 0;
		i = r * m.ld_mom + c;
		if (!again || !P.step || P.nesterov) load4(m.grad, r * m.ld_grad + c, P.type, wg, left, w);
		if (P.step) load4(again ? m.mom_out : m.mom, i, GL_F32, wm, left, v);
	};
	float kept[4][4];
	double sum = 0.0;
	for (unsigned e0 = threadIdx.x; e0 < total; e0 += 4 * SM_THREADS)
	{
		float w[4][4], v[4][4];
		long long i[4];
		int left[4];
		unsigned r, c;
#pragma unroll
		for (int k = 0; k < 4; ++k) fetch(e0 + k * SM_THREADS, false, w[k], v[k], i[k], left[k], r, c);
#pragma unroll
		for (int k = 0; k < 4; ++k)
		{
			if (P.step)
			{
#pragma unroll
				for (int j = 0; j < 4; ++j)
				{
					v[k][j] = fmaf(P.mu, v[k][j], w[k][j]);
					w[k][j] = P.nesterov ? fmaf(P.mu, v[k][j], w[k][j]) : v[k][j];
				}
				store4(m.mom_out, i[k], wm, left[k], v[k]);
			}
#pragma unroll
			for (int j = 0; j < 4; ++j)
			{
				sum = fma((double)w[k][j], (double)w[k][j], sum);
				if (e0 == threadIdx.x) kept[k][j] = w[k][j];
			}
		}
	}
	for (uint32_t i = threadIdx.x * 16; i < (uint32_t)(M.chunks * chunk); i += SM_THREADS * 16)
		*reinterpret_cast<uint4*>(gen + (xbase - base) + i) = make_uint4(0, 0, 0, 0);
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
	if (lane == 0) warp_sums[warp] = sum;
	asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
	__syncthreads();
	asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
	const uint32_t tmem_base = __shfl_sync(0xFFFFFFFFu, tmem_slot, 0);
	sum = 0.0;
	for (int w = 0; w <= SM_WARPS; ++w) sum += warp_sums[w];
	const double inv = inverse_norm(sum, P.eps);

	// ---- X_0: scaled, split, the short side as rows (every thread visits the elements that it has visited before)
	for (unsigned e0 = threadIdx.x; e0 < total; e0 += 4 * SM_THREADS)
	{
		float w[4][4], v[4][4];
		int left[4];
		unsigned r[4], c[4];
#pragma unroll
		for (int k = 0; k < 4; ++k)
		{
			long long i;
			if (e0 == threadIdx.x)
			{
				r[k] = (e0 + k * SM_THREADS) / quads;
				c[k] = (e0 + k * SM_THREADS - r[k] * quads) * 4;
				left[k] = e0 + k * SM_THREADS < total ? m.cols - (int)c[k] : 0;
#pragma unroll
				for (int j = 0; j < 4; ++j) w[k][j] = kept[k][j];
				continue;
			}
			fetch(e0 + k * SM_THREADS, true, w[k], v[k], i, left[k], r[k], c[k]);
#pragma unroll
			for (int j = 0; j < 4; ++j)
				if (P.step) w[k][j] = P.nesterov ? fmaf(P.mu, v[k][j], w[k][j]) : v[k][j];
		}
#pragma unroll
		for (int k = 0; k < 4; ++k)
		{
			if (left[k] <= 0) continue;
			float x[4];
#pragma unroll
			for (int j = 0; j < 4; ++j) x[j] = j < left[k] ? (float)((double)w[k][j] * inv) : 0.0f;
			uint2 h, l;
			split_pair(x[0], x[1], P.s0, h.x, l.x);
			split_pair(x[2], x[3], P.s0, h.y, l.y);
			if (!M.tall)
			{
				uint8_t* d = gen + (xbase - base) + c[k] / 64 * chunk + r[k] * 128 + (((c[k] / 8) ^ r[k]) & 7) * 16 + c[k] % 8 * 2;
				*reinterpret_cast<uint2*>(d) = h;
				*reinterpret_cast<uint2*>(d + part) = l;
				continue;
			}
#pragma unroll
			for (int j = 0; j < 4; ++j)
			{
				if (j >= left[k]) break;
				const unsigned i = c[k] + j;
				uint8_t* d = gen + (xbase - base) + r[k] / 64 * chunk + i * 128 + (((r[k] / 8) ^ i) & 7) * 16 + r[k] % 8 * 2;
				*reinterpret_cast<unsigned short*>(d) = (unsigned short)((j < 2 ? h.x : h.y) >> (16 * (j & 1)));
				*reinterpret_cast<unsigned short*>(d + part) = (unsigned short)((j < 2 ? l.x : l.y) >> (16 * (j & 1)));
			}
		}
	}
	asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
	__syncthreads();

	// ---- the products
	int buf = 0;         // next accumulator, and how often (mod 2) both have been used
	uint32_t ph = 0;
	bool ok = true;
	const int quarter = warp & 3, share = warp >> 2;  // epilogue: lanes of tensor memory, and every fourth eight columns
	const int row = quarter * 32 + lane;
	for (int n = 0; n < count; ++n)
	{
		const OrOp o = ops[n];
		const bool apply = o.b >= ID_X && o.a < ID_X;
		// 16-k steps: of X's columns (zeros behind the last), or of the short side
		const int steps = o.a >= ID_X ? 4 * M.chunks : rows / 16;
		// one accumulator takes SM_K steps of a square product, or two chunks of X
		const int turns = apply ? (M.chunks + 1) / 2 : (steps + SM_K - 1) / SM_K;
		if (warp == SM_WARPS)
		{
			const bool leader = elect_one();
			const uint32_t a = at(o.a), b = at(o.b);
			const uint64_t desc_a = make_smem_desc(a, 0u, 1024u, 2u);
			const uint64_t desc_b = make_smem_desc(b, apply ? (uint32_t)part : 0u, 1024u, 2u);
			const uint32_t a_low = (uint32_t)desc_a, a_high = (uint32_t)(desc_a >> 32), b_low = (uint32_t)desc_b, b_high = (uint32_t)(desc_b >> 32);
			const int width = apply ? 64 : rows;  // columns of an accumulator's half
			const uint32_t idesc = (1u << 4) | ((apply ? 1u : 0u) << 16) | ((uint32_t)(width >> 3) << 17) | ((uint32_t)(TC_BM >> 4) << 24);
			const uint32_t idesc2 = (1u << 4) | ((apply ? 1u : 0u) << 16) | ((uint32_t)(width >> 2) << 17) | ((uint32_t)(TC_BM >> 4) << 24);
			const uint32_t lo = (uint32_t)part >> 4, next = (uint32_t)chunk >> 4;
			for (int turn = 0; turn < turns && ok; ++turn)
			{
				ok = warp_wait(bar0 + 16 + 8 * buf, ph ^ 1u, abort_flag, P.status, 4);
				if (!ok) break;
				asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
				const uint32_t d = tmem_base + (uint32_t)(buf * SM_BUFFER);
				if (leader)
				{
					if (apply)
					{
						for (int c = 2 * turn; c < min(2 * turn + 2, M.chunks); ++c)
#pragma unroll 4
							for (int k = 0; k < steps; ++k)
							{
								// the first operand's k: chunk k / 4, 32 bytes per step; the second's: 16 rows of 128 bytes per step
								const uint32_t ak = a_low + (uint32_t)(k >> 2) * next + (uint32_t)(k & 3) * 2u, bk = b_low + (uint32_t)c * next + (uint32_t)k * 128u;
								mma(k == 0, d + (c & 1) * 128, ak, a_high, bk, b_high, idesc2);
								mma(false, d + (c & 1) * 128 + 64, ak + lo, a_high, bk, b_high, idesc);
							}
					}
					else
					{
#pragma unroll 4
						for (int k = turn * SM_K; k < min(steps, (turn + 1) * SM_K); ++k)
						{
							const uint32_t off = (uint32_t)(k >> 2) * next + (uint32_t)(k & 3) * 2u;
							mma(k == turn * SM_K, d, a_low + off, a_high, b_low + off, b_high, idesc2);
							mma(false, d + rows, a_low + lo + off, a_high, b_low + off, b_high, idesc);
						}
					}
					umma_commit(bar0 + 8 * buf);
				}
				__syncwarp();
				buf ^= 1;
				ph ^= (uint32_t)(buf == 0);
			}
		}
		else
		{
			float acc[4][8];
#pragma unroll
			for (int u = 0; u < 4; ++u)
#pragma unroll
				for (int i = 0; i < 8; ++i) acc[u][i] = 0.0f;
			for (int turn = 0; turn < turns && ok; ++turn)
			{
				// this warp's eights of columns: of the square result, or of the turn's two chunks
				const int eights = apply ? min(16, 8 * (M.chunks - 2 * turn)) : rows / 8;
				ok = warp_wait(bar0 + 8 * buf, ph, abort_flag, P.status, 3);
				if (!ok) break;
				asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
				if (quarter * 32 < rows)
				{
					const uint32_t d = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * SM_BUFFER);
#pragma unroll
					for (int u0 = 0; u0 < 4; u0 += 2)
					{
						uint32_t h[2][8], x[2][8];
						if (share + 4 * u0 >= eights) break;
#pragma unroll
						for (int u = 0; u < 2; ++u)
						{
							const int c8 = min(share + 4 * (u0 + u), eights - 1);  // (behind the last: loaded, not used)
							const uint32_t col = apply ? (uint32_t)((c8 >> 3) * 128 + (c8 & 7) * 8) : (uint32_t)(c8 * 8);
							tmem_ld8(d + col, h[u]);
							tmem_ld8(d + col + (apply ? 64 : rows), x[u]);
						}
						asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
						for (int u = 0; u < 2; ++u)
#pragma unroll
							for (int i = 0; i < 8; ++i) acc[u0 + u][i] = fmaf(o.f, __uint_as_float(h[u][i]), fmaf(o.f, __uint_as_float(x[u][i]), acc[u0 + u][i]));
					}
				}
				asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
				__syncwarp();
				if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar0 + 16 + 8 * buf) : "memory");
				buf ^= 1;
				ph ^= (uint32_t)(buf == 0);
				if (!apply && turn + 1 < turns) continue;
				if (row < rows)
				{
#pragma unroll
					for (int u = 0; u < 4; ++u)
					{
						const int c8 = share + 4 * u;
						if (c8 >= eights) break;
						const int j8 = apply ? 16 * turn + c8 : c8;  // eight of columns within the matrix
						const uint32_t off = (uint32_t)(j8 / 8 * chunk + row * 128 + ((j8 ^ row) & 7) * 16);
						float v[8];
#pragma unroll
						for (int i = 0; i < 8; ++i) v[i] = acc[u][i];
						auto add = [&](int id, float w) {
							if (id == ID_NONE) return;
							const uint8_t* e = gen + (at(id) - base) + off;
							const uint4 h4 = *reinterpret_cast<const uint4*>(e), l4 = *reinterpret_cast<const uint4*>(e + part);
							const __half2* hh = reinterpret_cast<const __half2*>(&h4);
							const __half2* ll = reinterpret_cast<const __half2*>(&l4);
#pragma unroll
							for (int i = 0; i < 4; ++i)
							{
								const float2 a2 = __half22float2(hh[i]), b2 = __half22float2(ll[i]);
								v[2 * i] = fmaf(w, a2.x + b2.x, v[2 * i]);
								v[2 * i + 1] = fmaf(w, a2.y + b2.y, v[2 * i + 1]);
							}
						};
						add(o.e, o.w);
						if (o.out != ID_NONE)
						{
							uint4 h4, l4;
							split_pair(v[0], v[1], o.so, h4.x, l4.x);
							split_pair(v[2], v[3], o.so, h4.y, l4.y);
							split_pair(v[4], v[5], o.so, h4.z, l4.z);
							split_pair(v[6], v[7], o.so, h4.w, l4.w);
							uint8_t* e = gen + (at(o.out) - base) + off;
							*reinterpret_cast<uint4*>(e) = h4;
							*reinterpret_cast<uint4*>(e + part) = l4;
						}
						else
						{
							// the result: the words' halves in the places of X's parts, for the pass that writes rows of the caller's matrix
							uint32_t hw[4], lw[4];
#pragma unroll
							for (int i = 0; i < 4; ++i)
							{
								const uint32_t b0 = __float_as_uint(v[2 * i]), b1 = __float_as_uint(v[2 * i + 1]);
								hw[i] = __byte_perm(b0, b1, 0x7632);
								lw[i] = __byte_perm(b0, b1, 0x5410);
							}
							uint8_t* e = gen + (xbase - base) + off;
							*reinterpret_cast<uint4*>(e) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
							*reinterpret_cast<uint4*>(e + part) = make_uint4(lw[0], lw[1], lw[2], lw[3]);
						}
					}
				}
#pragma unroll
				for (int u = 0; u < 4; ++u)
#pragma unroll
					for (int i = 0; i < 8; ++i) acc[u][i] = 0.0f;
			}
			asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
		}
		__syncthreads();
	}
	// ---- the result's rows: four neighbours per thread and turn again
	{
		const bool ww = P.step && (((uintptr_t)m.w | (uintptr_t)m.w_out | (uintptr_t)(m.ld_w * 4)) & 15) == 0;
		const bool wo = !P.step && (((uintptr_t)m.out | (uintptr_t)(m.ld_out * (P.type == GL_F32 ? 4 : 2))) & (P.type == GL_F32 ? 15 : 7)) == 0;
		const float keep = 1.0f - m.lr * P.decay;
		for (unsigned e0 = threadIdx.x; e0 < total; e0 += 4 * SM_THREADS)
		{
			float w[4][4];
#pragma unroll
			for (int k = 0; k < 4; ++k)
			{
				const unsigned e = e0 + k * SM_THREADS, r = e / quads, c = (e - r * quads) * 4;
				if (P.step) load4(m.w, r * m.ld_w + c, GL_F32, ww, e < total ? m.cols - (int)c : 0, w[k]);
			}
#pragma unroll
			for (int k = 0; k < 4; ++k)
			{
				const unsigned e = e0 + k * SM_THREADS, r = e / quads, c = (e - r * quads) * 4;
				if (e >= total) continue;
				const int left = m.cols - (int)c;
				float x[4];
				const uint8_t* d = gen + (xbase - base);
				if (!M.tall)
				{
					d += c / 64 * chunk + r * 128 + (((c / 8) ^ r) & 7) * 16 + c % 8 * 2;
					const uint2 h = *reinterpret_cast<const uint2*>(d), l = *reinterpret_cast<const uint2*>(d + part);
					x[0] = __uint_as_float(__byte_perm(l.x, h.x, 0x5410));
					x[1] = __uint_as_float(__byte_perm(l.x, h.x, 0x7632));
					x[2] = __uint_as_float(__byte_perm(l.y, h.y, 0x5410));
					x[3] = __uint_as_float(__byte_perm(l.y, h.y, 0x7632));
				}
				else
				{
#pragma unroll
					for (int j = 0; j < 4; ++j)
					{
						const unsigned i = min(c + j, (unsigned)m.cols - 1);
						const uint8_t* dj = d + r / 64 * chunk + i * 128 + (((r / 8) ^ i) & 7) * 16 + r % 8 * 2;
						x[j] = __uint_as_float((uint32_t)*reinterpret_cast<const unsigned short*>(dj) << 16 | *reinterpret_cast<const unsigned short*>(dj + part));
					}
				}
				if (P.step)
				{
#pragma unroll
					for (int j = 0; j < 4; ++j)
					{
						x[j] = fmaf(-m.lr, x[j], keep * w[k][j]);
						if (P.bad && j < left && !isfinite(x[j])) atomicOr(P.bad, 1);
					}
					store4(m.w_out, r * m.ld_w + c, ww, left, x);
				}
				else if (P.type == GL_F32) store4(static_cast<float*>(m.out), r * m.ld_out + c, wo, left, x);
				else
				{
#pragma unroll
					for (int j = 0; j < 4; ++j)
						if (j < left) store_typed(m.out, r * m.ld_out + c + j, x[j], P.type);
				}
			}
		}
	}
	if (*abort_flag && warp == SM_WARPS && lane == 0) mma_drain(bar0 + 32);
	asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
	__syncthreads();
	if (warp == SM_WARPS)
	{
		asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
		asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(SM_TMEM) : "memory");
	}
}

thread_local SmParams t_small;

// Shared memory of a matrix: A or R, X, and 128 rows from the last chunk's lo on.
size_t small_bytes(int p, int q)
{
	const int rows = (p + 15) / 16 * 16;
	const size_t part = small_part(rows);
	return ((rows + 63) / 64 + (size_t)(q + 63) / 64) * 2 * part + (size_t)(128 - rows) * 128 + 1024;
}

}  // namespace

bool ortho_small(int rows, int cols)
{
	const int p = std::min(rows, cols), q = std::max(rows, cols);
	// (2048: barriers, sums, operations.  Beyond 512 columns the many turns of one SM take longer than the rounds of many: 10 x 2048
	// 212 us a call)
	return p <= 128 && q <= 512 && small_bytes(p, q) <= SM_SMEM - 2048;
}

// (up to 1 << 17 elements, which take one CTA 130 us; 1 x 20000 in rounds of products takes 300.  Columns that move within their own
// memory are left to the kernels that read all of it first.)
bool ortho_vector(const OrthoMatrix& m)
{
	return std::min(m.rows, m.cols) == 1 && std::max(m.rows, m.cols) <= 1 << 17 && !(m.cols == 1 && m.out && m.out == m.grad && m.ld_out != m.ld_grad);
}

cudaError_t launch_ortho_small(const OrthoArgs& a, const OrProgram& prog, float s0, const OrthoMatrix* m, int count, int* status, bool reset, bool beside, cudaStream_t s)
{
	SmParams& P = t_small;
	P.prog = prog;
	P.count = count;
	P.type = a.type;
	P.step = a.step;
	P.nesterov = a.nesterov;
	P.reset = reset;
	P.mu = a.mu;
	P.decay = a.decay;
	P.eps = a.eps;
	P.bad = a.bad;
	P.s0 = s0;
	P.status = status;
	P.steps = a.steps;
	memcpy(P.coef, a.coef, sizeof P.coef);
	size_t smem = 0;
	for (int i = 0; i < count; ++i)
	{
		SmMat& M = P.mat[i];
		M.m = m[i];
		M.vector = ortho_vector(m[i]);
		M.p = std::min(M.m.rows, M.m.cols);
		M.q = std::max(M.m.rows, M.m.cols);
		M.tall = M.m.rows > M.m.cols;
		M.rows = (M.p + 15) / 16 * 16;
		M.chunks = (M.q + 63) / 64;
		if (!M.vector) smem = std::max(smem, small_bytes(M.p, M.q));
	}
	static_assert(sizeof(SmParams) < 32764, "kernel parameters");
	int sms = 0;
	if (cudaError_t e = prepare_tc_launch(reinterpret_cast<const void*>(&ortho_small_kernel), SM_SMEM - 2048, &sms)) return e;
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned)count);
	cfg.blockDim = dim3(SM_THREADS);
	cfg.dynamicSmemBytes = smem;
	cfg.stream = s;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	at[0].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = at;
	cfg.numAttrs = beside ? 1 : 0;
	return cudaLaunchKernelEx(&cfg, ortho_small_kernel, (const SmParams)P);
}

}  // namespace glb
