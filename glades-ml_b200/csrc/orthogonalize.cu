// Orthogonalisation of matrices by a polynomial iteration, and the weight update that is built on it.
//     X_0 = U / (|U|_F + eps),   A = X X^T,   P = a I + b A + c A^2,   X <- P X,   O = X_last
// drives the singular values of U towards 1 and keeps its singular vectors.  X is held with its short side p as rows (a tall
// matrix is transposed on the way in and on the way out), so that A and P are p x p.
//
// Bound: tensor cores.  Every product is fp32-faithful on three fp16 products (hi*hi + hi*lo + lo*hi), as the layer products of
// gemm_tcgen05.cu; unlike there the scales are known beforehand -- all singular values stay below a bound that follows from
// the coefficients alone -- so no product waits for a largest element, and lo is not scaled: the three products share one
// accumulator, tensor memory holds two of them, and the MMAs of one chunk run while the chunk in front is drained.  The
// error floor of an unscaled lo is 2^-25 of a unit, 2^-38 of the largest element.
// A and A^2 are symmetric: tiles above the diagonal are left out, an element below it is stored at both places.
//
// One cooperative launch walks all steps of all matrices: norm, scaling, then three phases per step, a grid barrier after
// each.  Within a phase every CTA takes the tiles cta, cta + grid, ... of all matrices.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "orthogonalize.h"
#include "tc_device.cuh"

namespace cg = cooperative_groups;

namespace glb {
using namespace tc;
namespace {

constexpr int OR_BK = 32;      // k per pipeline stage
// Stages whose products an accumulator takes before it is drained: the tensor core truncates as it adds, so a chain of n
// additions drifts by up to n * 2^-24 towards zero; 4 stages are 24 additions.
constexpr int OR_CHUNK = 4;
constexpr int OR_UNIT = 64;    // rows and columns of a piece of the elementwise phases

template <int BN>
struct OrSmem
{
	static constexpr int STAGES = BN == 256 ? 4 : (BN == 128 ? 6 : 8);
	static constexpr int EC = BN < 128 ? BN : 128;           // columns per epilogue warp
	static constexpr int EPI_WARPS = 4 * (BN / EC);
	static constexpr int THREADS = 64 + 32 * EPI_WARPS;
	static constexpr int A_BYTES = TC_BM * OR_BK * 2;
	static constexpr int B_BYTES = BN * OR_BK * 2;
	static constexpr int STAGE_BYTES = 2 * A_BYTES + 2 * B_BYTES;
	static constexpr int TILES_BYTES = STAGES * STAGE_BYTES;
	static constexpr int STAGING_BYTES = EPI_WARPS * 4096;   // at least a piece of the elementwise phases, 64 x 64 floats
	static constexpr int TOTAL = TILES_BYTES + STAGING_BYTES + 1024 /*alignment slack*/ + 512 /*barriers, sums*/;
};

struct OrMat
{
	OrthoMatrix m;
	int p, q, tall;
	long long ldx, planex;  // halfs: row pitch and size of one part of X; parts in the order X0 hi, X0 lo, X1 hi, X1 lo
	long long lds, planes;  // the same of A hi, A lo, P hi, P lo
	__half* X;
	__half* S;
	int units;              // pieces of the elementwise phases in front of this matrix's, and their number along a row
	int units_per_row;
};
struct OrMaps
{
	CUtensorMap xa, xb, xn, sa, sb;  // X as K-major A operand, K-major B operand, MN-major B operand; A and P as K-major operands
};
struct OrParams
{
	OrMaps maps[ORTHO_MAX_MATRICES];
	OrMat mat[ORTHO_MAX_MATRICES];
	int count, steps, units;
	int type, step, nesterov, reset;
	float mu, decay, eps;
	float coef[ORTHO_MAX_STEPS][3];
	int ex[ORTHO_MAX_STEPS + 1], ea[ORTHO_MAX_STEPS], ep[ORTHO_MAX_STEPS];  // exponents of the scales of X, A, P
	int* status;
	double* part;  // [matrix][grid] sums of squares
};

enum { PHASE_GRAM = 0, PHASE_POLY = 1, PHASE_APPLY = 2 };

// A phase's tiles of one matrix: rows m-tile by m-tile; of a symmetric product only the tiles that reach the diagonal.
__host__ __device__ inline int sym_tiles_of_row(int mt, int bn) { return (mt * TC_BM + TC_BM - 1) / bn + 1; }
__host__ __device__ inline int phase_tiles(int p, int q, int phase, int bn)
{
	const int tm = (p + TC_BM - 1) / TC_BM;
	if (phase == PHASE_APPLY) return tm * ((q + bn - 1) / bn);
	const int tn = (p + bn - 1) / bn;
	int n = 0;
	for (int mt = 0; mt < tm; ++mt)
	{
		const int c = sym_tiles_of_row(mt, bn);
		n += c < tn ? c : tn;
	}
	return n;
}

struct OrTile
{
	int mat, m0, n0, kb;
};
// tile t of a phase, or false
template <int BN>
__device__ __forceinline__ bool find_tile(const OrParams& P, int phase, int t, OrTile& o)
{
	for (int i = 0; i < P.count; ++i)
	{
		const int p = P.mat[i].p, q = P.mat[i].q;
		const int tm = (p + TC_BM - 1) / TC_BM;
		if (phase == PHASE_APPLY)
		{
			const int n = tm * ((q + BN - 1) / BN);
			if (t < n)
			{
				o.mat = i;
				o.m0 = (t % tm) * TC_BM;
				o.n0 = (t / tm) * BN;
				o.kb = (p + OR_BK - 1) / OR_BK;
				return true;
			}
			t -= n;
			continue;
		}
		const int tn = (p + BN - 1) / BN;
		for (int mt = tm - 1; mt >= 0; --mt)
		{
			const int n = min(tn, sym_tiles_of_row(mt, BN));
			if (t < n)
			{
				o.mat = i;
				o.m0 = mt * TC_BM;
				o.n0 = t * BN;
				o.kb = ((phase == PHASE_GRAM ? q : p) + OR_BK - 1) / OR_BK;
				return true;
			}
			t -= n;
		}
	}
	return false;
}

__device__ __forceinline__ float load_typed(const void* p, long long i, int type)
{
	if (type == GL_F32) return static_cast<const float*>(p)[i];
	if (type == GL_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
	return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_typed(void* p, long long i, float v, int type)
{
	if (type == GL_F32) static_cast<float*>(p)[i] = v;
	else if (type == GL_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
	else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// What element (r, c) contributes: the gradient itself, or the momentum that it makes (left in mom_out by the first visit).
__device__ __forceinline__ float first_visit(const OrParams& P, const OrthoMatrix& m, int r, int c)
{
	const float g = load_typed(m.grad, (long long)r * m.ld_grad + c, P.type);
	if (!P.step) return g;
	const long long i = (long long)r * m.ld_mom + c;
	const float v = fmaf(P.mu, m.mom[i], g);
	m.mom_out[i] = v;
	return P.nesterov ? fmaf(P.mu, v, g) : v;
}
__device__ __forceinline__ float second_visit(const OrParams& P, const OrthoMatrix& m, int r, int c)
{
	if (!P.step) return load_typed(m.grad, (long long)r * m.ld_grad + c, P.type);
	const float v = m.mom_out[(long long)r * m.ld_mom + c];
	return P.nesterov ? fmaf(P.mu, v, load_typed(m.grad, (long long)r * m.ld_grad + c, P.type)) : v;
}

// hi and lo of x * s, lo unscaled
__device__ __forceinline__ void split_plain(float x, float s, __half& hi, __half& lo)
{
	const float xs = x * s;
	hi = __float2half_rn(xs);
	lo = __float2half_rn(xs - __half2float(hi));
}
__device__ __forceinline__ void split_pair(float x, float y, float s, uint32_t& hi, uint32_t& lo)
{
	const float xs = x * s, ys = y * s;
	const __half2 h = __floats2half2_rn(xs, ys);
	const float2 f = __half22float2(h);
	const __half2 l = __floats2half2_rn(xs - f.x, ys - f.y);
	hi = *reinterpret_cast<const uint32_t*>(&h);
	lo = *reinterpret_cast<const uint32_t*>(&l);
}

// 32 x 32 piece, a row per lane: as the rows of a matrix of parts.  Through shared memory, eight rows of 64 bytes per access.
__device__ __forceinline__ void store_rows(const float (&v)[32], float s, __half* hi, __half* lo, long long ld, uint32_t area, int lane)
{
	__syncwarp();
#pragma unroll
	for (int k = 0; k < 4; ++k)
	{
		uint32_t h[4], l[4];
#pragma unroll
		for (int i = 0; i < 4; ++i) split_pair(v[8 * k + 2 * i], v[8 * k + 2 * i + 1], s, h[i], l[i]);
		const uint32_t row = area + (uint32_t)lane * 128u;
		asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + (uint32_t)((k ^ (lane & 7)) << 4)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
		asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + (uint32_t)(((k + 4) ^ (lane & 7)) << 4)), "r"(l[0]), "r"(l[1]), "r"(l[2]), "r"(l[3]) : "memory");
	}
	__syncwarp();
#pragma unroll
	for (int i = 0; i < 8; ++i)
	{
		const int r = i * 4 + (lane >> 3), k = lane & 7;
		uint4 w;
		asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(area + (uint32_t)r * 128u + (uint32_t)((k ^ (r & 7)) << 4)));
		__half* d = (k < 4 ? hi : lo) + (long long)r * ld + (k & 3) * 8;
		*reinterpret_cast<uint4*>(d) = w;
	}
}
// the same piece transposed: column j is row j of the destination
__device__ __forceinline__ void store_columns(const float (&v)[32], float s, __half* hi, __half* lo, long long ld, int lane)
{
#pragma unroll
	for (int j = 0; j < 32; ++j)
	{
		__half h, l;
		split_plain(v[j], s, h, l);
		hi[(long long)j * ld + lane] = h;
		lo[(long long)j * ld + lane] = l;
	}
}
// 32 x 32 floats in shared memory, element (r, c) at r * 32 + (c ^ r): rows and columns without bank conflicts
__device__ __forceinline__ uint32_t square_at(uint32_t area, int r, int c) { return area + (uint32_t)((r * 32 + (c ^ r)) * 4); }
__device__ __forceinline__ void square_put(uint32_t area, int r, int c, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(square_at(area, r, c)), "f"(v) : "memory"); }
__device__ __forceinline__ float square_get(uint32_t area, int r, int c)
{
	float v;
	asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(square_at(area, r, c)) : "memory");
	return v;
}

template <int BN>
__global__ void __launch_bounds__(OrSmem<BN>::THREADS, 1) ortho_kernel(const __grid_constant__ OrParams P)
{
	using S = OrSmem<BN>;
	constexpr int STAGES = S::STAGES, EC = S::EC, THREADS = S::THREADS;
	extern __shared__ uint8_t smem_raw[];
	const uint32_t raw = smem_u32(smem_raw);
	const uint32_t base = (raw + 1023u) & ~1023u;
	uint8_t* gen_base = smem_raw + (base - raw);
	const uint32_t staging0 = base + S::TILES_BYTES;
	float* piece = reinterpret_cast<float*>(gen_base + S::TILES_BYTES);  // the elementwise phases' 64 x 64 piece
	const uint32_t bar0 = staging0 + S::STAGING_BYTES;
	// barrier slots: full[s] = s, empty[s] = STAGES + s, acc_full[2], acc_empty[2], given_up
	constexpr int NBARS = 2 * STAGES + 5;
	const uint32_t bar_acc_full = bar0 + 8 * (2 * STAGES), bar_acc_empty = bar_acc_full + 16, bar_given_up = bar_acc_full + 32;
	uint8_t* tail = gen_base + S::TILES_BYTES + S::STAGING_BYTES + 8 * NBARS;
	uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail);
	volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 4);
	double* warp_sums = reinterpret_cast<double*>(tail + 8);  // 10 at most

	cg::grid_group grid = cg::this_grid();
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

	if (threadIdx.x == 0)
	{
		for (int s = 0; s < STAGES; ++s)
		{
			mbar_init(bar0 + 8 * s, 1);
			mbar_init(bar0 + 8 * (STAGES + s), 1);
		}
		for (int b = 0; b < 2; ++b)
		{
			mbar_init(bar_acc_full + 8 * b, 1);
			mbar_init(bar_acc_empty + 8 * b, S::EPI_WARPS);
		}
		mbar_init(bar_given_up, 1);
		*abort_flag = 0;
		asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
		if (blockIdx.x == 0 && P.reset) *P.status = 0;  // (nothing can raise it before the first grid barrier)
	}
	if (warp == 1)
	{
		asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * BN) : "memory");
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
	}
	asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
	__syncthreads();
	asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
	const uint32_t tmem_base = *tmem_slot;

	// ---- sums of squares, in double (a product of two floats is exact there and does not leave its range)
	for (int i = 0; i < P.count; ++i)
	{
		const OrMat& M = P.mat[i];
		const int units = M.units_per_row * ((M.m.rows + OR_UNIT - 1) / OR_UNIT);
		double sum = 0.0;
		// (unit u of matrix i belongs to CTA (M.units + u) mod grid, here and in the next phase)
		const int first = ((int)blockIdx.x - M.units % (int)gridDim.x + (int)gridDim.x) % (int)gridDim.x;
		for (int u = first; u < units; u += gridDim.x)
		{
			const int r0 = (u / M.units_per_row) * OR_UNIT, c0 = (u % M.units_per_row) * OR_UNIT;
#pragma unroll 4
			for (int e = threadIdx.x; e < OR_UNIT * OR_UNIT; e += THREADS)
			{
				const int r = r0 + e / OR_UNIT, c = c0 + e % OR_UNIT;
				if (r < M.m.rows && c < M.m.cols)
				{
					const double v = first_visit(P, M.m, r, c);
					sum = fma(v, v, sum);
				}
			}
		}
#pragma unroll
		for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
		__syncthreads();
		if (lane == 0) warp_sums[warp] = sum;
		__syncthreads();
		if (threadIdx.x == 0)
		{
			double t = 0.0;
			for (int w = 0; w < THREADS / 32; ++w) t += warp_sums[w];
			P.part[i * gridDim.x + blockIdx.x] = t;
		}
	}
	grid.sync();

	// ---- X_0: scaled, split, the short side as rows
	for (int i = 0; i < P.count; ++i)
	{
		const OrMat& M = P.mat[i];
		const int units = M.units_per_row * ((M.m.rows + OR_UNIT - 1) / OR_UNIT);
		const int first = ((int)blockIdx.x - M.units % (int)gridDim.x + (int)gridDim.x) % (int)gridDim.x;
		if (first >= units) continue;
		if (warp == 0)
		{
			double t = 0.0;
			for (int k = lane; k < (int)gridDim.x; k += 32) t += P.part[i * gridDim.x + k];
#pragma unroll
			for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
			if (lane == 0) warp_sums[0] = t;
		}
		__syncthreads();
		const float norm = (float)sqrt(warp_sums[0]) + P.eps;
		const float s = pow2f(P.ex[0]);
		__syncthreads();
		for (int u = first; u < units; u += gridDim.x)
		{
			const int r0 = (u / M.units_per_row) * OR_UNIT, c0 = (u % M.units_per_row) * OR_UNIT;
#pragma unroll 4
			for (int e = threadIdx.x; e < OR_UNIT * OR_UNIT; e += THREADS)
			{
				const int rr = e / OR_UNIT, cc = e % OR_UNIT;
				const int r = r0 + rr, c = c0 + cc;
				if (r < M.m.rows && c < M.m.cols)
				{
					const float x = second_visit(P, M.m, r, c) / norm;
					if (M.tall) piece[rr * OR_UNIT + (cc ^ (rr & 31))] = x;
					else
					{
						__half h, l;
						split_plain(x, s, h, l);
						M.X[r * M.ldx + c] = h;
						M.X[M.planex + r * M.ldx + c] = l;
					}
				}
			}
			if (M.tall)
			{
				__syncthreads();
#pragma unroll 4
				for (int e = threadIdx.x; e < OR_UNIT * OR_UNIT; e += THREADS)
				{
					const int cc = e / OR_UNIT, rr = e % OR_UNIT;
					const int r = r0 + rr, c = c0 + cc;
					if (r < M.m.rows && c < M.m.cols)
					{
						__half h, l;
						split_plain(piece[rr * OR_UNIT + (cc ^ (rr & 31))], s, h, l);
						M.X[c * M.ldx + r] = h;
						M.X[M.planex + c * M.ldx + r] = l;
					}
				}
				__syncthreads();
			}
		}
	}
	asm volatile("fence.proxy.async;" ::: "memory");  // (the copies read through another proxy what ordinary stores have written)
	grid.sync();

	// ---- the products
	int s = 0;             // producer, MMA lane: next stage, and how often (mod 2) the ring has been walked
	uint32_t ph = 0;
	int issued = 0;
	int buf = 0;           // MMA lane, epilogue: next accumulator, and how often (mod 2) both have been used
	uint32_t aph = 0;
	bool ok = true;
	const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
	const int half = (warp - 2) >> 2;
	for (int step = 0; step < P.steps; ++step)
	{
		const int cur = step & 1;
		for (int phase = PHASE_GRAM; phase <= PHASE_APPLY; ++phase)
		{
			OrTile t;
			if (warp == 0 && lane == 0)
			{
				// ------------------------------------------------ TMA producer
				asm volatile("fence.proxy.async;" ::: "memory");
				for (int ti = blockIdx.x; ok && find_tile<BN>(P, phase, ti, t); ti += gridDim.x)
				{
					const OrMaps& mp = P.maps[t.mat];
					const int plane_a = phase == PHASE_GRAM ? 2 * cur : (phase == PHASE_POLY ? 0 : 2);
					const CUtensorMap* ma = phase == PHASE_GRAM ? &mp.xa : &mp.sa;
					for (int kb = 0; kb < t.kb; ++kb)
					{
						const uint32_t full = bar0 + 8 * s;
						if (!mbar_wait(full + 8 * STAGES, ph ^ 1u, abort_flag, P.status, 1))
						{
							ok = false;
							break;
						}
						mbar_expect_tx(full, S::STAGE_BYTES);
						const uint32_t sa = base + s * S::STAGE_BYTES;
						tma_load_3d(sa, ma, full, kb * OR_BK, t.m0, plane_a);
						if (phase == PHASE_APPLY) tma_load_4d(sa + 2 * S::A_BYTES, &mp.xn, full, 0, kb * OR_BK, t.n0 / 64, 2 * cur);
						else if (phase == PHASE_GRAM) tma_load_3d(sa + 2 * S::A_BYTES, &mp.xb, full, kb * OR_BK, t.n0, 2 * cur);
						else tma_load_3d(sa + 2 * S::A_BYTES, &mp.sb, full, kb * OR_BK, t.n0, 0);
						++issued;
						if (++s == STAGES)
						{
							s = 0;
							ph ^= 1u;
						}
					}
				}
			}
			else if (warp == 1 && lane == 0)
			{
				// ------------------------------------------------ MMA issuer (layouts and descriptors: gemm_tcgen05.cu)
				const uint32_t b_mn = phase == PHASE_APPLY ? 1u : 0u;
				const uint32_t idesc = (1u << 4) | (b_mn << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(TC_BM >> 4) << 24);
				const uint64_t desc_a = make_smem_desc(base, 0u, 512u, 4u);
				const uint64_t desc_b = make_smem_desc(base + 2 * S::A_BYTES, b_mn ? 128u * OR_BK : 0u, b_mn ? 1024u : 512u, b_mn ? 2u : 4u);
				const uint32_t a_step = 32u >> 4, b_step = b_mn ? 2048u >> 4 : 32u >> 4;
				constexpr uint32_t A_LO = S::A_BYTES >> 4, B_LO = S::B_BYTES >> 4;
				for (int ti = blockIdx.x; ok && find_tile<BN>(P, phase, ti, t); ti += gridDim.x)
				{
					int in = 0;
					for (int left = t.kb; left > 0; --left)
					{
						if (in == 0)
						{
							if (!mbar_wait(bar_acc_empty + 8 * buf, aph ^ 1u, abort_flag, P.status, 4)) { ok = false; break; }
						}
						const uint32_t full = bar0 + 8 * s;
						if (!mbar_wait(full, ph, abort_flag, P.status, 2)) { ok = false; break; }
						asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
						const uint32_t off = (uint32_t)s * (S::STAGE_BYTES >> 4);
						const uint64_t a0 = desc_a + off, b0 = desc_b + off;
						const uint64_t a1 = a0 + a_step, b1 = b0 + b_step;
						const uint32_t d = tmem_base + (uint32_t)(buf * BN);
						umma_f16(d, a0, b0 + B_LO, idesc, (uint32_t)in);
						umma_f16(d, a0 + A_LO, b0, idesc, 1u);
						umma_f16(d, a1, b1 + B_LO, idesc, 1u);
						umma_f16(d, a1 + A_LO, b1, idesc, 1u);
						umma_f16(d, a0, b0, idesc, 1u);
						umma_f16(d, a1, b1, idesc, 1u);
						umma_commit(full + 8 * STAGES);
						if (++in == OR_CHUNK || left == 1)
						{
							umma_commit(bar_acc_full + 8 * buf);
							in = 0;
							buf ^= 1;
							aph ^= (uint32_t)(buf == 0);
						}
						if (++s == STAGES)
						{
							s = 0;
							ph ^= 1u;
						}
					}
				}
			}
			else if (warp >= 2)
			{
				// ------------------------------------------------ epilogue
				const bool last = phase == PHASE_APPLY && step == P.steps - 1;
				const int es = phase == PHASE_GRAM ? 2 * P.ex[step] : (phase == PHASE_POLY ? 2 * P.ea[step] : P.ep[step] + P.ex[step]);
				const float inv = pow2f(-es);
				const float so = pow2f(phase == PHASE_GRAM ? P.ea[step] : (phase == PHASE_POLY ? P.ep[step] : P.ex[step + 1]));
				const uint32_t area = staging0 + (uint32_t)(warp - 2) * 4096u;
				for (int ti = blockIdx.x; ok && find_tile<BN>(P, phase, ti, t); ti += gridDim.x)
				{
					const OrMat& M = P.mat[t.mat];
					float acc[EC];
#pragma unroll
					for (int i = 0; i < EC; ++i) acc[i] = 0.0f;
					for (int done = 0; done < t.kb; done += OR_CHUNK)
					{
						if (!mbar_wait(bar_acc_full + 8 * buf, aph, abort_flag, P.status, 3))
						{
							ok = false;
							break;
						}
						asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
						const uint32_t taddr = tmem_base + lane_base + (uint32_t)(buf * BN + half * EC);
#pragma unroll
						for (int c = 0; c < EC / 16; ++c)
						{
							uint32_t r[16];
							tmem_ld16(taddr + (uint32_t)(c * 16), r);
							asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
							for (int e = 0; e < 16; ++e) acc[c * 16 + e] += __uint_as_float(r[e]);
						}
						asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
						__syncwarp();
						if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_acc_empty + 8 * buf) : "memory");
						buf ^= 1;
						aph ^= (uint32_t)(buf == 0);
					}
					if (!ok) break;
					const int r0 = t.m0 + (warp & 3) * 32;
					if (r0 >= M.p) continue;
#pragma unroll
					for (int pc = 0; pc < EC / 32; ++pc)
					{
						const int c0 = t.n0 + half * EC + pc * 32;
						float v[32];
#pragma unroll
						for (int i = 0; i < 32; ++i) v[i] = acc[pc * 32 + i] * inv;
						if (phase == PHASE_APPLY)
						{
							if (c0 >= M.q) continue;
							if (!last)
							{
								__half* X = M.X + 2 * (cur ^ 1) * M.planex + (long long)r0 * M.ldx + c0;
								store_rows(v, so, X, X + M.planex, M.ldx, area, lane);
								continue;
							}
							const OrthoMatrix& m = M.m;
							const float keep = 1.0f - m.lr * P.decay;
							__syncwarp();
							if (!M.tall)
							{
#pragma unroll
								for (int j = 0; j < 32; ++j) square_put(area, lane, j, v[j]);
								__syncwarp();
							}
							// row j of the piece (column j of a tall matrix's), one element per lane
#pragma unroll
							for (int j = 0; j < 32; ++j)
							{
								const int r = M.tall ? c0 + j : r0 + j, c = M.tall ? r0 + lane : c0 + lane;
								if (r >= m.rows || c >= m.cols) continue;
								const float o = M.tall ? v[j] : square_get(area, j, lane);
								if (!P.step) store_typed(m.out, r * m.ld_out + c, o, P.type);
								else
								{
									const long long i = r * m.ld_w + c;
									m.w_out[i] = fmaf(-m.lr, o, keep * m.w[i]);
								}
							}
							continue;
						}
						// a symmetric result: what lies above the diagonal is another tile's mirror image
						if (c0 > r0) continue;
						__half* out = M.S + (phase == PHASE_POLY ? 2 * M.planes : 0);
						if (phase == PHASE_POLY)
						{
							const float b = P.coef[step][1], c = P.coef[step][2], ia = pow2f(-P.ea[step]);
							const __half* A = M.S + (long long)(r0 + lane) * M.lds + c0;
#pragma unroll
							for (int k = 0; k < 4; ++k)
							{
								const uint4 h4 = *reinterpret_cast<const uint4*>(A + 8 * k);
								const uint4 l4 = *reinterpret_cast<const uint4*>(A + M.planes + 8 * k);
								const __half2* h = reinterpret_cast<const __half2*>(&h4);
								const __half2* l = reinterpret_cast<const __half2*>(&l4);
#pragma unroll
								for (int i = 0; i < 4; ++i)
								{
									const float2 x = __half22float2(h[i]), y = __half22float2(l[i]);
									v[8 * k + 2 * i] = fmaf(c, v[8 * k + 2 * i], b * ((x.x + y.x) * ia));
									v[8 * k + 2 * i + 1] = fmaf(c, v[8 * k + 2 * i + 1], b * ((x.y + y.y) * ia));
								}
							}
						}
						if (c0 == r0)
						{
							// on the diagonal: the upper half becomes the lower half's mirror image
							__syncwarp();
#pragma unroll
							for (int j = 0; j < 32; ++j) square_put(area, lane, j, v[j]);
							__syncwarp();
#pragma unroll
							for (int j = 0; j < 32; ++j)
							{
								if (j > lane) v[j] = square_get(area, j, lane);
								if (j == lane && phase == PHASE_POLY) v[j] += P.coef[step][0];
							}
						}
						__half* D = out + (long long)r0 * M.lds + c0;
						store_rows(v, so, D, D + M.planes, M.lds, area, lane);
						if (c0 != r0)
						{
							__half* T = out + (long long)c0 * M.lds + r0;
							store_columns(v, so, T, T + M.planes, M.lds, lane);
						}
					}
				}
				asm volatile("fence.proxy.async;" ::: "memory");
			}
			if (!(phase == PHASE_APPLY && step == P.steps - 1)) grid.sync();
		}
	}
	if (*abort_flag)
	{
		// copies that are still in flight are given a bounded time to land, and so are the MMAs
		if (warp == 0 && lane == 0) mbar_drain<STAGES>(bar0, issued > STAGES ? issued - STAGES : 0, issued);
		if (warp == 1 && lane == 0) mma_drain(bar_given_up);
	}
	asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
	__syncthreads();
	if (warp == 1)
	{
		asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
		asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * BN) : "memory");
	}
}

// ---- host ----------------------------------------------------------------------------------------------------
constexpr size_t OR_HEADER = 256;  // status word
constexpr int OR_SMS = 148;
constexpr size_t OR_PART = (size_t)ORTHO_MAX_MATRICES * OR_SMS * sizeof(double);
size_t round_up(size_t v, size_t m) { return (v + m - 1) / m * m; }

size_t matrix_bytes(int rows, int cols)
{
	const size_t p = round_up((size_t)std::min(rows, cols), 128), q = round_up((size_t)std::max(rows, cols), 128);
	return (4 * p * q + 4 * p * p) * sizeof(__half);
}

// 2^e * bound < 2^15
int exponent_for(double bound)
{
	int e = 0;
	frexp(bound, &e);  // bound < 2^e
	return std::min(15 - e, 40);
}

template <int BN>
bool make_maps(OrMaps& o, const OrMat& M)
{
	auto map3 = [&](CUtensorMap* m, const __half* base, long long rows, long long cols, long long ld, long long plane, int box_rows) {
		return tc_make_parts_map(m, base, rows, cols, ld, plane, 4, OR_BK, box_rows);
	};
	return map3(&o.xa, M.X, M.p, M.q, M.ldx, M.planex, TC_BM) && map3(&o.xb, M.X, M.p, M.q, M.ldx, M.planex, BN) &&
	       tc_make_parts_map_mn(&o.xn, M.X, M.p, M.q, M.ldx, M.planex, 4, OR_BK, BN) &&
	       map3(&o.sa, M.S, M.p, M.p, M.lds, M.planes, TC_BM) && map3(&o.sb, M.S, M.p, M.p, M.lds, M.planes, BN);
}

// About how many clocks the products take: for each phase the CTA with the most work.  A k-block's six MMAs cost 768 clocks
// on 256 columns, 400 on 128 and 300 on 64 (where reading A from shared memory bounds them), a tile about 2500 more.
long long estimate(const OrParams& P, int bn)
{
	const long long per = bn == 256 ? 768 : (bn == 128 ? 400 : 300);
	long long total = 0;
	for (int phase = 0; phase < 3; ++phase)
	{
		long long load[OR_SMS] = {0}, worst = 0;
		int t = 0;
		for (int i = 0; i < P.count; ++i)
		{
			const int n = phase_tiles(P.mat[i].p, P.mat[i].q, phase, bn);
			const long long kb = ((phase == PHASE_GRAM ? P.mat[i].q : P.mat[i].p) + OR_BK - 1) / OR_BK;
			// (whole rounds at once, the rest one by one)
			const long long rounds = n / OR_SMS;
			for (int c = 0; c < OR_SMS && rounds; ++c) load[c] += rounds * (kb * per + 2500);
			for (int k = 0; k < n % OR_SMS; ++k) load[(t + k) % OR_SMS] += kb * per + 2500;
			t = (t + n) % OR_SMS;
		}
		for (long long l : load) worst = std::max(worst, l);
		total += worst;
	}
	return total;
}

template <int BN>
cudaError_t launch_width(OrParams& P, int grid_most, cudaStream_t s)
{
	for (int i = 0; i < P.count; ++i)
		if (!make_maps<BN>(P.maps[i], P.mat[i])) return cudaErrorInvalidValue;
	int sms = 0;
	cudaError_t e = prepare_tc_launch(reinterpret_cast<const void*>(ortho_kernel<BN>), OrSmem<BN>::TOTAL, &sms);
	if (e != cudaSuccess) return e;
	int most = 1;
	for (int phase = 0; phase < 3; ++phase)
	{
		int n = 0;
		for (int i = 0; i < P.count; ++i) n += phase_tiles(P.mat[i].p, P.mat[i].q, phase, BN);
		most = std::max(most, n);
	}
	most = std::max(most, P.units);
	int grid = std::min(std::min(sms, grid_most), most);
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned)grid);
	cfg.blockDim = dim3(OrSmem<BN>::THREADS);
	cfg.dynamicSmemBytes = OrSmem<BN>::TOTAL;
	cfg.stream = s;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeCooperative;
	at[0].val.cooperative = 1;
	cfg.attrs = at;
	cfg.numAttrs = 1;
	return cudaLaunchKernelEx(&cfg, ortho_kernel<BN>, (const OrParams)P);
}

}  // namespace

bool ortho_bounds(const float (*coef)[3], int steps, double* sx, double* sa, double* sp)
{
	// the largest singular value that a step may find, by the extrema of the step's polynomial on [0, largest]
	sx[0] = 1.0 + 1e-5;  // (the norm's rounding)
	for (int k = 0; k < steps; ++k)
	{
		const double a = coef[k][0], b = coef[k][1], c = coef[k][2], t = sx[k];
		if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
		sa[k] = t * t * (1.0 + 1e-5);
		auto h = [&](double l) { return fabs(a + l * (b + l * c)); };  // P's eigenvalue for A's eigenvalue l
		sp[k] = std::max(h(0.0), h(sa[k]));
		if (c != 0.0 && -b / (2 * c) > 0.0 && -b / (2 * c) < sa[k]) sp[k] = std::max(sp[k], h(-b / (2 * c)));
		double most = h(t * t) * t;
		// a + 3 b l + 5 c l^2 = 0 with l = s^2
		double roots[2];
		int n = 0;
		if (c != 0.0)
		{
			const double d = 9 * b * b - 20 * a * c;
			if (d >= 0.0)
			{
				roots[n++] = (-3 * b + sqrt(d)) / (10 * c);
				roots[n++] = (-3 * b - sqrt(d)) / (10 * c);
			}
		}
		else if (b != 0.0) roots[n++] = -a / (3 * b);
		for (int i = 0; i < n; ++i)
			if (roots[i] > 0.0 && roots[i] < t * t) most = std::max(most, h(roots[i]) * sqrt(roots[i]));
		sx[k + 1] = most * (1.0 + 1e-4);
		if (!(sx[k + 1] <= 16.0) || !(sp[k] <= 256.0)) return false;
	}
	return true;
}

size_t ortho_workspace_bytes(const OrthoMatrix* m, int count)
{
	size_t most = 0;
	for (int first = 0; first < count; first += ORTHO_MAX_MATRICES)
	{
		size_t b = 0;
		for (int i = first; i < std::min(count, first + ORTHO_MAX_MATRICES); ++i) b += matrix_bytes(m[i].rows, m[i].cols);
		most = std::max(most, b);
	}
	return 256 + OR_HEADER + round_up(OR_PART, 256) + most;  // (256: the caller's pointer need not be aligned)
}

int* ortho_status(void* work) { return reinterpret_cast<int*>(round_up((size_t)work, 256)); }

cudaError_t launch_orthogonalize(const OrthoArgs& a, void* work, cudaStream_t s)
{
	char* w = reinterpret_cast<char*>(ortho_status(work));
	double sx[ORTHO_MAX_STEPS + 1], sa[ORTHO_MAX_STEPS], sp[ORTHO_MAX_STEPS];
	if (!ortho_bounds(a.coef, a.steps, sx, sa, sp)) return cudaErrorInvalidValue;
	for (int first = 0; first < a.count; first += ORTHO_MAX_MATRICES)
	{
		static thread_local OrParams P;
		memset(&P, 0, sizeof P);
		P.count = std::min(ORTHO_MAX_MATRICES, a.count - first);
		P.steps = a.steps;
		P.type = a.type;
		P.step = a.step;
		P.nesterov = a.nesterov;
		P.mu = a.mu;
		P.decay = a.decay;
		P.eps = a.eps;
		P.reset = first == 0;
		P.status = a.status ? a.status : reinterpret_cast<int*>(w);
		if (a.status) P.reset = 0;
		P.part = reinterpret_cast<double*>(w + OR_HEADER);
		for (int k = 0; k < a.steps; ++k)
		{
			for (int j = 0; j < 3; ++j) P.coef[k][j] = a.coef[k][j];
			P.ea[k] = exponent_for(sa[k]);
			P.ep[k] = exponent_for(sp[k]);
		}
		for (int k = 0; k <= a.steps; ++k) P.ex[k] = exponent_for(sx[k]);
		char* at = w + OR_HEADER + round_up(OR_PART, 256);
		for (int i = 0; i < P.count; ++i)
		{
			OrMat& M = P.mat[i];
			M.m = a.mat[first + i];
			M.tall = M.m.rows > M.m.cols;
			M.p = std::min(M.m.rows, M.m.cols);
			M.q = std::max(M.m.rows, M.m.cols);
		}
		// the matrices with the longest products first: what is left for the last CTAs of a phase is small
		std::stable_sort(P.mat, P.mat + P.count, [](const OrMat& x, const OrMat& y) { return (double)x.p * x.q > (double)y.p * y.q; });
		for (int i = 0; i < P.count; ++i)
		{
			OrMat& M = P.mat[i];
			M.ldx = (long long)round_up(M.q, 128);
			M.planex = M.ldx * (long long)round_up(M.p, 128);
			M.lds = (long long)round_up(M.p, 128);
			M.planes = M.lds * M.lds;
			M.X = reinterpret_cast<__half*>(at);
			M.S = M.X + 4 * M.planex;
			at += matrix_bytes(M.m.rows, M.m.cols);
			M.units = P.units;
			M.units_per_row = (M.m.cols + OR_UNIT - 1) / OR_UNIT;
			P.units += M.units_per_row * ((M.m.rows + OR_UNIT - 1) / OR_UNIT);
		}
		const long long c64 = estimate(P, 64), c128 = estimate(P, 128), c256 = estimate(P, 256);
		cudaError_t e;
		if (c256 <= c128 && c256 <= c64) e = launch_width<256>(P, OR_SMS, s);
		else if (c128 <= c64) e = launch_width<128>(P, OR_SMS, s);
		else e = launch_width<64>(P, OR_SMS, s);
		if (e != cudaSuccess) return e;
	}
	return cudaSuccess;
}

}  // namespace glb
