// Orthogonalisation of matrices by a polynomial iteration, and the weight update that is built on it.
//     X_0 = U / (|U|_F + eps),   A = X X^T,   R = b A + c A^2,   X <- a X + R X,   O = X_last
// drives the singular values of U towards 1 and keeps its singular vectors.  X is held with its short side p as rows (a tall
// matrix is transposed on the way in and on the way out), so that A and R are p x p.
//
// Multiply-adds of a step: p^2 q / 2 (A) + p^3 / 2 (A A), which are symmetric, and p^2 q.
// (Several steps on the short side alone -- P = a + R commutes with A, so that the next step's A is P A P and X needs one product for
// all of them -- take half of the multiply-adds of a flat matrix.  But the rounding of A is absolute, and small singular values lose
// digits with every further step: 512 x 4096 came out up to 5 times further off than with fp32 products.)
//
// Bound: tensor cores.  Every product is fp32-faithful on three fp16 products (hi*hi + hi*lo + lo*hi), as the layer products of
// gemm_tcgen05.cu; unlike there the scales are known beforehand -- all singular values stay below a bound that follows from
// the coefficients alone -- so no product waits for a largest element, and lo is not scaled (its error floor is 2^-25 of a unit,
// 2^-38 of the largest element): tensor memory holds two accumulators of a tile, and the MMAs of one chunk run while the
// chunk in front is drained.  hi and lo of the second operand lie one behind the other in shared memory and are one operand of
// twice the columns, [hi*hi | hi*lo], an accumulator for each half: two MMAs per 16 k instead of three, fewer reads of shared memory.
// (Tiles of 256 columns, which only fit with one accumulator for all three products, lost: their epilogue holds 128 sums per
// thread, spills, and the MMAs wait for it.  4096 x 4096, a step: 769 us against 655.)
// a X (or b A) is where the epilogue's registers start from, loaded while the first chunk is computed: inside the accumulator
// it would be truncated with every addition, which doubles the error of the result.  The products are multiplied by their own
// coefficient as they are added, so that every coefficient is used as it is given.
// A and R are symmetric: tiles above the diagonal are left out, an element below it is stored at both places.
//
// One cooperative launch walks all steps of all matrices: norm, scaling, then a round for each product of the program, of all
// matrices at once, a grid barrier after each.  Within a round every CTA takes the items cta, cta + grid, ... of all matrices.  Where a
// round has too few tiles for the SMs, its tiles are split along k: the parts go to scratch in fp32, and after one more
// barrier all warps of the GPU add them up, 32 x 32 elements at a time, in a fixed order.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "ortho_device.cuh"

namespace cg = cooperative_groups;

namespace glb {
using namespace tc;
namespace {

static_assert(OR_BM == TC_BM, "tiles");
constexpr int OR_UNIT = 64;    // rows and columns of a piece of the elementwise phases
constexpr int OR_SMS = 148;
constexpr int OR_SQUARES = 2;  // p x p matrices of parts: A and R
constexpr int OR_SPLIT_K = 128; // k that a part of a split tile has at least
// An accumulator takes one stage, four additions, before it is drained.  The tensor core truncates as it adds: a sum of one sign loses
// half a unit in the last place with every addition, and the polynomial multiplies an error that all singular values share by up to 15.
// Against 64 bits, relative to the error of fp32 products, with 8 additions -> 4: random 256 x 1000 1.4 -> 0.8, 256 x 256 with near singular
// values 1.6 -> 1.0, 192 x 192 with orthogonal rows 2.5 -> 1.5, for 1 to 6 % of the time.  (What is lost cannot be put back by a factor:
// sums that cancel, or of few products, lose less.  A factor that made up for it on random matrices left diagonal and block diagonal
// ones 4 times further off than fp32 products.)

template <int BN>
struct OrSmem
{
	static constexpr int COLUMNS = 2 * BN;                   // of an accumulator
	static constexpr int STAGES = BN == 128 ? 3 : 4;
	static constexpr int EC = BN / 2;                        // columns per epilogue warp
	static constexpr int EPI_WARPS = 8;
	static constexpr int FIRST = 4;                          // epilogue warps 4 ..; 0 copies, 1 multiplies, 2 and 3 help with elementwise work
	static constexpr int THREADS = 32 * (FIRST + EPI_WARPS);
	static constexpr int A_BYTES = TC_BM * OR_BK * 2;
	static constexpr int B_BYTES = BN * OR_BK * 2;
	static constexpr int STAGE_BYTES = 2 * A_BYTES + 2 * B_BYTES;
	static constexpr int TILES_BYTES = STAGES * STAGE_BYTES;
	static constexpr int STAGING_BYTES = EPI_WARPS * 4096;   // at least a piece of the elementwise phases, 64 x 64 floats
	static constexpr int PIECES = 4 * (BN / 32);             // 32 x 32 pieces of a tile
	static constexpr int TOTAL = TILES_BYTES + STAGING_BYTES + 1024 /*alignment slack*/ + 512 /*barriers, sums*/;
};

struct OrMat
{
	OrthoMatrix m;
	int p, q, tall;
	long long ldx, planex;  // halfs: row pitch and size of one part of X; parts in the order X0 hi, X0 lo, X1 hi, X1 lo
	long long lds, planes;  // the same of the p x p matrices
	__half* X;
	__half* S;
	int units;              // pieces of the elementwise phases in front of this matrix's, and their number along a row
	int units_per_row;
};
struct OrMaps
{
	CUtensorMap xa, xb, xn, sa, sb;  // X as K-major A operand, K-major B operand, MN-major B operand; p x p as K-major operands
};
struct OrParams
{
	OrMaps maps[ORTHO_MAX_MATRICES];
	OrMat mat[ORTHO_MAX_MATRICES];
	OrProgram prog;  // operation k is round k's, of every matrix
	unsigned char split[ORTHO_MAX_MATRICES][OR_MAX_OPS];
	unsigned long long reduce;  // rounds with split tiles
	int items[OR_MAX_OPS], splits[OR_MAX_OPS];  // a round's items, and its split tiles
	int count, units;
	int type, step, nesterov, reset;
	float mu, decay, eps, s0;  // s0: X_0's scale
	int* status;
	int* bad;
	unsigned* arrived;  // CTAs at the rounds' barriers
	double* sums;  // [matrix][grid] sums of squares
	float4* part;  // parts of split tiles
};

// ---- 32 x 32 pieces, a row per lane --------------------------------------------------------------------------------
// 16-byte chunk k (0 .. 3 hi, 4 .. 7 lo) of row r in the warp's staging area
__device__ __forceinline__ uint32_t chunk_at(uint32_t area, int r, int k) { return area + (uint32_t)(r * 128 + ((k ^ (r & 7)) << 4)); }
// the parts of v * s into the staging area
__device__ __forceinline__ void stage_parts(const float (&v)[32], float s, uint32_t area, int lane)
{
	__syncwarp();
#pragma unroll
	for (int k = 0; k < 4; ++k)
	{
		uint32_t h[4], l[4];
#pragma unroll
		for (int i = 0; i < 4; ++i) split_pair(v[8 * k + 2 * i], v[8 * k + 2 * i + 1], s, h[i], l[i]);
		asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk_at(area, lane, k)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
		asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk_at(area, lane, k + 4)), "r"(l[0]), "r"(l[1]), "r"(l[2]), "r"(l[3]) : "memory");
	}
	__syncwarp();
}
// the staged piece as rows of a matrix of parts, four rows of 64 bytes of hi and of lo per access
__device__ __forceinline__ void store_staged(__half* hi, long long plane, long long ld, uint32_t area, int lane)
{
	const int k = lane & 7;
	__half* d = hi + (k < 4 ? 0 : plane) + (long long)(lane >> 3) * ld + (k & 3) * 8;
	uint4 w[8];
#pragma unroll
	for (int i = 0; i < 8; ++i)
		asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w) : "r"(chunk_at(area, i * 4 + (lane >> 3), k)));
#pragma unroll
	for (int i = 0; i < 8; ++i)
	{
		*reinterpret_cast<uint4*>(d) = w[i];
		d += 4 * ld;
	}
}
// The staged piece transposed in place, 8 x 8 elements at a time: lane l gives the address of row l % 8 of block l / 8 of four.
__device__ __forceinline__ void transpose_staged(uint32_t area, int lane)
{
	uint32_t w[8][4];
	const int b = lane >> 3, r = lane & 7;
	// blocks (4 rows of blocks) x (4 columns of hi, 4 of lo): one access takes a column of blocks
#pragma unroll
	for (int k = 0; k < 8; ++k)
		asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
		             : "=r"(w[k][0]), "=r"(w[k][1]), "=r"(w[k][2]), "=r"(w[k][3])
		             : "r"(chunk_at(area, b * 8 + r, k)));
	__syncwarp();
	// block (i, k) becomes block (k, i) of its part
#pragma unroll
	for (int k = 0; k < 8; ++k)
		asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(chunk_at(area, (k & 3) * 8 + r, (k & 4) + b)),
		             "r"(w[k][0]), "r"(w[k][1]), "r"(w[k][2]), "r"(w[k][3])
		             : "memory");
	__syncwarp();
}
// acc += w * (32 elements of row r from column c on of the matrix of parts id)
__device__ __forceinline__ void add_parts(float* acc, float w, int id, const OrMat& M, int r, int c)
{
	if (id == ID_NONE) return;
	const long long plane = id >= ID_X ? M.planex : M.planes;
	const __half* hi = id >= ID_X ? M.X + 2 * (id - ID_X) * plane + r * M.ldx + c : M.S + 2 * id * plane + r * M.lds + c;
#pragma unroll
	for (int k = 0; k < 4; ++k)
	{
		const uint4 h4 = *reinterpret_cast<const uint4*>(hi + 8 * k);
		const uint4 l4 = *reinterpret_cast<const uint4*>(hi + plane + 8 * k);
		const __half2* h = reinterpret_cast<const __half2*>(&h4);
		const __half2* l = reinterpret_cast<const __half2*>(&l4);
#pragma unroll
		for (int i = 0; i < 4; ++i)
		{
			const float2 x = __half22float2(h[i]), y = __half22float2(l[i]);
			acc[8 * k + 2 * i] = fmaf(w, x.x + y.x, acc[8 * k + 2 * i]);
			acc[8 * k + 2 * i + 1] = fmaf(w, x.y + y.y, acc[8 * k + 2 * i + 1]);
		}
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
// v: column per lane
__device__ __forceinline__ void transpose(float (&v)[32], uint32_t area, int lane)
{
	__syncwarp();
#pragma unroll
	for (int j = 0; j < 32; ++j) square_put(area, lane, j, v[j]);
	__syncwarp();
#pragma unroll
	for (int j = 0; j < 32; ++j) v[j] = square_get(area, j, lane);
}

// the result's elements of column (tall: row) c0 + lane ... of the caller's matrix: v[j] is element (r + j, c) of it
template <int TYPE>
__device__ __forceinline__ void store_result(const float (&v)[32], void* out, long long ld, int r, int c, int rows, int cols)
{
	if (c >= cols) return;
	const int n = rows - r;
	const long long i = r * ld + c;
#pragma unroll
	for (int j = 0; j < 32; ++j)
		if (j < n)
		{
			if (TYPE == GL_F32) static_cast<float*>(out)[i + j * ld] = v[j];
			else if (TYPE == GL_BF16) static_cast<__nv_bfloat16*>(out)[i + j * ld] = __float2bfloat16_rn(v[j]);
			else static_cast<__half*>(out)[i + j * ld] = __float2half_rn(v[j]);
		}
}
__device__ __forceinline__ void update_weights(const float (&v)[32], const OrthoMatrix& m, float decay, int* bad, int r, int c)
{
	bool finite = true;
	if (c >= m.cols) return;
	const int n = m.rows - r;
	const float keep = 1.0f - m.lr * decay;
	const float* w = m.w + r * m.ld_w + c;
	float* o = m.w_out + r * m.ld_w + c;
#pragma unroll
	for (int b = 0; b < 32; b += 16)
	{
		float x[16];
#pragma unroll
		for (int j = 0; j < 16; ++j) x[j] = b + j < n ? w[(b + j) * m.ld_w] : 0.0f;
#pragma unroll
		for (int j = 0; j < 16; ++j)
			if (b + j < n)
			{
				const float y = fmaf(-m.lr, v[b + j], keep * x[j]);
				finite = finite && isfinite(y);
				o[(b + j) * m.ld_w] = y;
			}
	}
	if (bad && !finite) atomicOr(bad, 1);
}

// What the epilogue needs of an operation and its matrix, asked for before the products are awaited: the parameters lie in
// constant memory, whose first touch takes as long as a copy from L2.
struct OrTarget
{
	float so;
	int kind, p, q;  // kind: 0 the caller's matrix, 1 symmetric, 2 X
	__half* D;
	long long plane, ld;
	__device__ __forceinline__ OrTarget(const OrMat& M, const OrOp& o)
	{
		so = o.so;
		p = M.p;
		q = M.q;
		kind = op_symmetric(o) ? 1 : (o.out == ID_NONE ? 0 : 2);
		plane = o.out >= ID_X ? M.planex : M.planes;
		ld = o.out >= ID_X ? M.ldx : M.lds;
		D = o.out >= ID_X ? M.X + 2 * (o.out - ID_X) * plane : M.S + 2 * (o.out < 0 ? 0 : o.out) * plane;
		asm volatile("" : "+f"(so), "+r"(p), "+r"(q), "+r"(kind), "+l"(plane), "+l"(ld), "+l"(D));
	}
	// pieces that lie outside the matrix, or above the diagonal of a symmetric result (another piece's mirror image)
	__device__ __forceinline__ bool needs(int r0, int c0) const { return r0 < p && (kind == 1 ? c0 <= r0 : c0 < q); }
};
// what becomes of a piece of a product: rows r0 + lane, columns c0 ..
__device__ __forceinline__ void finish_piece(const OrParams& P, int mat, const OrTarget& T, float (&v)[32], int r0, int c0, uint32_t area, int lane)
{
	if (T.kind == 0)
	{
		const OrMat& M = P.mat[mat];
		if (!M.tall) transpose(v, area, lane);
		// a wide matrix: lane = column, v = rows r0 ..; a tall one is transposed already: lane = its column, v = its rows c0 ..
		const int r = M.tall ? c0 : r0, c = (M.tall ? r0 : c0) + lane;
		if (P.step) update_weights(v, M.m, P.decay, P.bad, r, c);
		else if (P.type == GL_F32) store_result<GL_F32>(v, M.m.out, M.m.ld_out, r, c, M.m.rows, M.m.cols);
		else if (P.type == GL_BF16) store_result<GL_BF16>(v, M.m.out, M.m.ld_out, r, c, M.m.rows, M.m.cols);
		else store_result<GL_F16>(v, M.m.out, M.m.ld_out, r, c, M.m.rows, M.m.cols);
		return;
	}
	if (T.kind == 1 && c0 == r0)
	{
		// on the diagonal: the upper half becomes the lower half's mirror image
		__syncwarp();
#pragma unroll
		for (int j = 0; j < 32; ++j) square_put(area, lane, j, v[j]);
		__syncwarp();
#pragma unroll
		for (int j = 0; j < 32; ++j)
			if (j > lane) v[j] = square_get(area, j, lane);
	}
	stage_parts(v, T.so, area, lane);
	store_staged(T.D + (long long)r0 * T.ld + c0, T.plane, T.ld, area, lane);
	if (T.kind == 1 && c0 != r0)
	{
		__syncwarp();
		transpose_staged(area, lane);
		store_staged(T.D + (long long)c0 * T.ld + r0, T.plane, T.ld, area, lane);
	}
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32])
{
	asm volatile(
	    "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
	    "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
	    "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
	    : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
	      "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
	      "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
	      "=r"(r[31])
	    : "r"(taddr)
	    : "memory");
}

// The grid barrier: CTAs count themselves without waiting for the count, and then watch it (the cooperative launch has
// them all resident; against the runtime's barrier it saves a way to L2 and back: 256 x 256, 15 rounds, 110 -> 106 us).  Bounded:
// false where a CTA has not come.
constexpr int MEETING_LOST = 2;
__device__ __forceinline__ bool meet(unsigned* arrived, unsigned all, volatile int* abort_flag, int* err_flag)
{
	__syncthreads();
	if (threadIdx.x == 0)
	{
		asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(arrived) : "memory");
		const long long t0 = clock64();
		for (;;)
		{
			unsigned v;
			asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(arrived) : "memory");
			if (v >= all) break;
			if (clock64() - t0 > 8 * TC_WAIT_CYCLES)  // (a CTA may have to sit out its own waits)
			{
				*abort_flag = MEETING_LOST;
				atomicExch(err_flag, 5);
				break;
			}
		}
	}
	__syncthreads();
	return *abort_flag != MEETING_LOST;
}

// A warp has been asked for an item that its round does not have.
__device__ __noinline__ static void give_up(volatile int* abort_flag, int* err_flag, int lane)
{
	if (lane != 0) return;
	*abort_flag = 1;
	atomicExch(err_flag, 6);
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
	double* warp_sums = reinterpret_cast<double*>(tail + 8);  // one per warp

	cg::grid_group grid = cg::this_grid();
	cudaTriggerProgrammaticLaunchCompletion();  // (single rows and columns have nothing to wait for)
	const int warp = __shfl_sync(0xFFFFFFFFu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

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
		// (nothing can raise the one before the first grid barrier, which is the runtime's, nor count on the other)
		if (blockIdx.x == 0 && P.reset) *P.status = 0;
		if (blockIdx.x == 0) *P.arrived = 0;
	}
	if (warp == 1)
	{
		asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * S::COLUMNS) : "memory");
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
	}
	asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
	__syncthreads();
	asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
	const uint32_t tmem_base = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);

	// ---- the elementwise phases: pieces of 64 x 64 elements; piece u of matrix i belongs to CTA (M.units + u) mod grid in both.
	// Four neighbours per thread and turn, the loads of all its turns ahead of the stores.
	constexpr int QUADS = OR_UNIT * OR_UNIT / 4;
	constexpr int TURNS = (QUADS + THREADS - 1) / THREADS;
	auto wide_ok = [](const void* p, long long ld, int size) { return (((uintptr_t)p | (uintptr_t)(ld * size)) & (4 * size - 1)) == 0; };
	// sums of squares, in double (a product of two floats is exact there and does not leave its range)
	for (int i = 0; i < P.count; ++i)
	{
		const OrMat& M = P.mat[i];
		const OrthoMatrix& m = M.m;
		const bool wg = wide_ok(m.grad, m.ld_grad, P.type == GL_F32 ? 4 : 2);
		const bool wm = P.step && wide_ok(m.mom, m.ld_mom, 4) && wide_ok(m.mom_out, m.ld_mom, 4);
		const int units = M.units_per_row * ((m.rows + OR_UNIT - 1) / OR_UNIT);
		double sum = 0.0;
		const int first = ((int)blockIdx.x - M.units % (int)gridDim.x + (int)gridDim.x) % (int)gridDim.x;
		for (int u = first; u < units; u += gridDim.x)
		{
			const int r0 = (u / M.units_per_row) * OR_UNIT, c0 = (u % M.units_per_row) * OR_UNIT;
			float g[TURNS][4], v[TURNS][4];
#pragma unroll
			for (int k = 0; k < TURNS; ++k)
			{
				const int e = threadIdx.x + k * THREADS;
				const int r = r0 + e / (OR_UNIT / 4), c = c0 + e % (OR_UNIT / 4) * 4;
				const int left = e < QUADS && r < m.rows ? m.cols - c : 0;
				load4(m.grad, (long long)r * m.ld_grad + c, P.type, wg, left, g[k]);
				if (P.step) load4(m.mom, (long long)r * m.ld_mom + c, GL_F32, wm, left, v[k]);
			}
#pragma unroll
			for (int k = 0; k < TURNS; ++k)
			{
				if (P.step)
				{
					const int e = threadIdx.x + k * THREADS;
					const int r = r0 + e / (OR_UNIT / 4), c = c0 + e % (OR_UNIT / 4) * 4;
					const int left = e < QUADS && r < m.rows ? m.cols - c : 0;
#pragma unroll
					for (int j = 0; j < 4; ++j)
					{
						v[k][j] = fmaf(P.mu, v[k][j], g[k][j]);
						g[k][j] = P.nesterov ? fmaf(P.mu, v[k][j], g[k][j]) : v[k][j];
					}
					store4(m.mom_out, (long long)r * m.ld_mom + c, wm, left, v[k]);
				}
#pragma unroll
				for (int j = 0; j < 4; ++j) sum = fma((double)g[k][j], (double)g[k][j], sum);
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
			P.sums[i * gridDim.x + blockIdx.x] = t;
		}
	}
	grid.sync();

	// X_0: scaled, split, the short side as rows
	for (int i = 0; i < P.count; ++i)
	{
		const OrMat& M = P.mat[i];
		const OrthoMatrix& m = M.m;
		const bool wg = wide_ok(m.grad, m.ld_grad, P.type == GL_F32 ? 4 : 2);
		const bool wm = P.step && wide_ok(m.mom_out, m.ld_mom, 4);
		const int units = M.units_per_row * ((m.rows + OR_UNIT - 1) / OR_UNIT);
		const int first = ((int)blockIdx.x - M.units % (int)gridDim.x + (int)gridDim.x) % (int)gridDim.x;
		if (first >= units) continue;
		if (warp == 0)
		{
			double t = 0.0;
			for (int k = lane; k < (int)gridDim.x; k += 32) t += P.sums[i * gridDim.x + k];
#pragma unroll
			for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
			if (lane == 0) warp_sums[0] = t;
		}
		__syncthreads();
		const double inv = inverse_norm(warp_sums[0], P.eps);
		const float s = P.s0;
		__syncthreads();
		for (int u = first; u < units; u += gridDim.x)
		{
			const int r0 = (u / M.units_per_row) * OR_UNIT, c0 = (u % M.units_per_row) * OR_UNIT;
			float g[TURNS][4], v[TURNS][4];
#pragma unroll
			for (int k = 0; k < TURNS; ++k)
			{
				const int e = threadIdx.x + k * THREADS;
				const int r = r0 + e / (OR_UNIT / 4), c = c0 + e % (OR_UNIT / 4) * 4;
				const int left = e < QUADS && r < m.rows ? m.cols - c : 0;
				if (!P.step || P.nesterov) load4(m.grad, (long long)r * m.ld_grad + c, P.type, wg, left, g[k]);
				if (P.step) load4(m.mom_out, (long long)r * m.ld_mom + c, GL_F32, wm, left, v[k]);
			}
#pragma unroll
			for (int k = 0; k < TURNS; ++k)
			{
				const int e = threadIdx.x + k * THREADS;
				const int rr = e / (OR_UNIT / 4), cc = e % (OR_UNIT / 4) * 4;
				const int r = r0 + rr, c = c0 + cc;
				if (e >= QUADS || r >= m.rows || c >= m.cols) continue;
				float x[4];
#pragma unroll
				for (int j = 0; j < 4; ++j)
				{
					const float w = !P.step ? g[k][j] : (P.nesterov ? fmaf(P.mu, v[k][j], g[k][j]) : v[k][j]);
					x[j] = (float)((double)w * inv);
				}
				if (M.tall)
				{
#pragma unroll
					for (int j = 0; j < 4; ++j) piece[rr * OR_UNIT + ((cc + j) ^ (rr & 31))] = x[j];
				}
				else
				{
					// (what lies beyond the last column is never read)
					uint2 h, l;
					split_pair(x[0], x[1], s, h.x, l.x);
					split_pair(x[2], x[3], s, h.y, l.y);
					*reinterpret_cast<uint2*>(M.X + r * M.ldx + c) = h;
					*reinterpret_cast<uint2*>(M.X + M.planex + r * M.ldx + c) = l;
				}
			}
			if (M.tall)
			{
				__syncthreads();
#pragma unroll
				for (int k = 0; k < 2 * TURNS; ++k)
				{
					// two rows of the matrix (columns of X) per thread and turn, neighbouring lanes neighbouring pairs
					const int e = threadIdx.x + k * THREADS;
					const int cc = e / (OR_UNIT / 2), rr = e % (OR_UNIT / 2) * 2;
					const int r = r0 + rr, c = c0 + cc;
					if (cc >= OR_UNIT || r >= m.rows || c >= m.cols) continue;
					uint32_t h, l;
					split_pair(piece[rr * OR_UNIT + (cc ^ (rr & 31))], piece[(rr + 1) * OR_UNIT + (cc ^ ((rr + 1) & 31))], s, h, l);
					*reinterpret_cast<uint32_t*>(M.X + c * M.ldx + r) = h;
					*reinterpret_cast<uint32_t*>(M.X + M.planex + c * M.ldx + r) = l;
				}
				__syncthreads();
			}
		}
	}
	unsigned meeting = gridDim.x;
	const bool met = meet(P.arrived, meeting, abort_flag, P.status);

	// ---- the products
	int s = 0;             // producer, MMA warp: next stage, and how often (mod 2) the ring has been walked
	uint32_t ph = 0;
	int issued = 0;
	int buf = 0;           // MMA warp, epilogue: next accumulator, and how often (mod 2) both have been used
	uint32_t aph = 0;
	bool ok = true;
	OrItem t;              // copying and multiplying warps: a round's first item is looked up in front of the barrier before it
	auto look_up = [&](int round, int ti) {
		if (find_item<BN>(P, round, ti, t)) return true;
		give_up(abort_flag, P.status, lane);
		return false;
	};
	if (warp < 2 && (int)blockIdx.x < P.items[0]) ok = look_up(0, blockIdx.x);
	for (int round = 0; met && round < P.prog.count; ++round)
	{
		const int items = P.items[round];
		const OrOp& o = P.prog.op[round];
		if (warp == 0)
		{
			// ------------------------------------------------ TMA producer
			// (the copies read through another proxy what ordinary stores of all CTAs have written to global memory in front of the grid
			// barrier; a fence for all state spaces costs 0.45 us more in every round)
			asm volatile("fence.proxy.async.global;" ::: "memory");
			const bool leader = elect_one();
			for (int ti = blockIdx.x; ok && ti < items; ti += gridDim.x)
			{
				if (ti != (int)blockIdx.x && !look_up(round, ti)) { ok = false; break; }
				const OrMaps& mp = P.maps[t.mat];
				const bool ax = o.a >= ID_X, bx = o.b >= ID_X;
				const CUtensorMap* ma = ax ? &mp.xa : &mp.sa;
				const CUtensorMap* mb = ax ? &mp.xb : &mp.sb;
				const int pa = 2 * (ax ? o.a - ID_X : o.a), pb = 2 * (bx ? o.b - ID_X : o.b);
				const bool mn = bx && !ax;
				for (int kb = t.kb0; kb < t.kb1; ++kb)
				{
					const uint32_t full = bar0 + 8 * s;
					if (!warp_wait(full + 8 * STAGES, ph ^ 1u, abort_flag, P.status, 1))
					{
						ok = false;
						break;
					}
					if (leader)
					{
						mbar_expect_tx(full, S::STAGE_BYTES);
						const uint32_t sa = base + s * S::STAGE_BYTES;
						tma_load_3d(sa, ma, full, kb * OR_BK, t.m0, pa);
						if (mn) tma_load_4d(sa + 2 * S::A_BYTES, &mp.xn, full, 0, kb * OR_BK, t.n0 / 64, pb);
						else tma_load_3d(sa + 2 * S::A_BYTES, mb, full, kb * OR_BK, t.n0, pb);
					}
					__syncwarp();
					++issued;
					if (++s == STAGES)
					{
						s = 0;
						ph ^= 1u;
					}
				}
			}
		}
		else if (warp == 1)
		{
			// ------------------------------------------------ MMA issuer (layouts and descriptors: gemm_tcgen05.cu)
			const bool leader = elect_one();
			for (int ti = blockIdx.x; ok && ti < items; ti += gridDim.x)
			{
				if (ti != (int)blockIdx.x && !look_up(round, ti)) { ok = false; break; }
				const uint32_t b_mn = o.b >= ID_X && o.a < ID_X ? 1u : 0u;
				const uint32_t idesc = (1u << 4) | (b_mn << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(TC_BM >> 4) << 24);
				const uint32_t idesc2 = (1u << 4) | (b_mn << 16) | ((uint32_t)(S::COLUMNS >> 3) << 17) | ((uint32_t)(TC_BM >> 4) << 24);
				// K-major: rows of 128 bytes, eight of them a group; MN-major: 64 columns by OR_BK k; 128-byte swizzle
				const uint64_t desc_a = make_smem_desc(base, 0u, 1024u, 2u);
				const uint64_t desc_b = make_smem_desc(base + 2 * S::A_BYTES, b_mn ? 128u * OR_BK : 0u, 1024u, 2u);
				const uint32_t a_low = (uint32_t)desc_a, a_high = (uint32_t)(desc_a >> 32), b_low = (uint32_t)desc_b, b_high = (uint32_t)(desc_b >> 32);
				const uint32_t a_step = 32u >> 4, b_step = b_mn ? 2048u >> 4 : 32u >> 4;
				constexpr uint32_t A_LO = S::A_BYTES >> 4;
				for (int left = t.kb1 - t.kb0; left > 0; --left)
				{
					if (!warp_wait(bar_acc_empty + 8 * buf, aph ^ 1u, abort_flag, P.status, 4)) { ok = false; break; }
					const uint32_t full = bar0 + 8 * s;
					if (!warp_wait(full, ph, abort_flag, P.status, 2)) { ok = false; break; }
					asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
					const uint32_t off = (uint32_t)s * (S::STAGE_BYTES >> 4);
					const uint32_t a0 = a_low + off, b0 = b_low + off;
					const uint32_t d = tmem_base + (uint32_t)(buf * S::COLUMNS);
					if (leader)
					{
#pragma unroll
						for (int k = 0; k < OR_BK / 16; ++k)
						{
							mma(k == 0, d, a0 + k * a_step, a_high, b0 + k * b_step, b_high, idesc2);
							mma(false, d + BN, a0 + A_LO + k * a_step, a_high, b0 + k * b_step, b_high, idesc);
						}
						umma_commit(full + 8 * STAGES);
						umma_commit(bar_acc_full + 8 * buf);
					}
					__syncwarp();
					buf ^= 1;
					aph ^= (uint32_t)(buf == 0);
					if (++s == STAGES)
					{
						s = 0;
						ph ^= 1u;
					}
				}
			}
		}
		else if (warp >= S::FIRST)
		{
			// ------------------------------------------------ epilogue
			const uint32_t area = staging0 + (uint32_t)(warp - S::FIRST) * 4096u;
			const int quarter = warp & 3, half = (warp - S::FIRST) >> 2;
			for (int ti = blockIdx.x; ok && ti < items; ti += gridDim.x)
			{
				if (!look_up(round, ti)) { ok = false; break; }
				const OrMat& M = P.mat[t.mat];
				const OrTarget target(M, o);
				const float f = o.f;
				const int r0 = t.m0 + quarter * 32, c00 = t.n0 + half * EC;
				float acc[EC];
#pragma unroll
				for (int i = 0; i < EC; ++i) acc[i] = 0.0f;
				if (t.kb0 == 0)
				{
#pragma unroll
					for (int pc = 0; pc < EC / 32; ++pc)
						if (target.needs(r0, c00 + pc * 32)) add_parts(acc + pc * 32, o.w, o.e, M, r0 + lane, c00 + pc * 32);
				}
				for (int left = t.kb1 - t.kb0; left > 0; --left)
				{
					if (!warp_wait(bar_acc_full + 8 * buf, aph, abort_flag, P.status, 3))
					{
						ok = false;
						break;
					}
					asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
					const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * S::COLUMNS + half * EC);
#pragma unroll
					for (int c = 0; c < EC / 32; ++c)
#pragma unroll
						for (int h = 1; h >= 0; --h)
						{
							uint32_t r[32];
							tmem_ld32(taddr + (uint32_t)(h * BN + c * 32), r);
							asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
							for (int e = 0; e < 32; ++e) acc[c * 32 + e] = fmaf(f, __uint_as_float(r[e]), acc[c * 32 + e]);
						}
					asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
					__syncwarp();
					if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_acc_empty + 8 * buf) : "memory");
					buf ^= 1;
					aph ^= (uint32_t)(buf == 0);
				}
				if (!ok) break;
#pragma unroll
				for (int pc = 0; pc < EC / 32; ++pc)
				{
					const int c0 = c00 + pc * 32;
					if (!target.needs(r0, c0)) continue;
					if (t.split > 1)
					{
						float4* d = P.part + ((long long)t.slot * S::PIECES + quarter * (BN / 32) + half * (EC / 32) + pc) * 256 + lane;
#pragma unroll
						for (int j = 0; j < 8; ++j)
							d[j * 32] = make_float4(acc[pc * 32 + 4 * j], acc[pc * 32 + 4 * j + 1], acc[pc * 32 + 4 * j + 2], acc[pc * 32 + 4 * j + 3]);
						continue;
					}
					float v[32];
#pragma unroll
					for (int i = 0; i < 32; ++i) v[i] = acc[pc * 32 + i];
					finish_piece(P, t.mat, target, v, r0, c0, area, lane);
				}
			}
		}
		if (P.reduce >> round & 1)
		{
			if (!meet(P.arrived, meeting += gridDim.x, abort_flag, P.status)) break;
			if (warp >= S::FIRST)
			{
				const uint32_t area = staging0 + (uint32_t)(warp - S::FIRST) * 4096u;
				const int warps = (int)gridDim.x * S::EPI_WARPS;
				// (neighbouring pieces on different SMs)
				for (int k = (warp - S::FIRST) * (int)gridDim.x + (int)blockIdx.x; k < P.splits[round] * S::PIECES; k += warps)
				{
					if (!find_split<BN>(P, round, k / S::PIECES, t))
					{
						give_up(abort_flag, P.status, lane);
						break;
					}
					const OrTarget target(P.mat[t.mat], o);
					const int pc = k % S::PIECES;
					const int r0 = t.m0 + pc / (BN / 32) * 32, c0 = t.n0 + pc % (BN / 32) * 32;
					if (!target.needs(r0, c0)) continue;
					float v[32];
					const float4* d = P.part + ((long long)t.slot * S::PIECES + pc) * 256 + lane;
#pragma unroll
					for (int j = 0; j < 8; ++j)
					{
						const float4 x = d[j * 32];
						v[4 * j] = x.x; v[4 * j + 1] = x.y; v[4 * j + 2] = x.z; v[4 * j + 3] = x.w;
					}
#pragma unroll 2
					for (int part = 1; part < t.split; ++part)
					{
						d += S::PIECES * 256;
#pragma unroll
						for (int j = 0; j < 8; ++j)
						{
							const float4 x = d[j * 32];
							v[4 * j] += x.x; v[4 * j + 1] += x.y; v[4 * j + 2] += x.z; v[4 * j + 3] += x.w;
						}
					}
					finish_piece(P, t.mat, target, v, r0, c0, area, lane);
				}
			}
		}
		if (round + 1 < P.prog.count)
		{
			if (ok && warp < 2 && (int)blockIdx.x < P.items[round + 1]) ok = look_up(round + 1, blockIdx.x);
			if (!meet(P.arrived, meeting += gridDim.x, abort_flag, P.status)) break;
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
		asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * S::COLUMNS) : "memory");
	}
}

// ---- host ----------------------------------------------------------------------------------------------------
constexpr size_t OR_HEADER = 256;  // status word; half of it further the barriers' count
constexpr size_t OR_SUMS = (size_t)ORTHO_MAX_MATRICES * OR_SMS * sizeof(double);
size_t round_up(size_t v, size_t m) { return (v + m - 1) / m * m; }

struct Bounds
{
	double sx[ORTHO_MAX_STEPS + 1];  // singular values of X before a step
	double sa[ORTHO_MAX_STEPS];      // eigenvalues of A,
	double sr[ORTHO_MAX_STEPS];      // of R = b A + c A^2
};
// The largest singular value that a step may find follows from the extrema of its polynomial on [0, largest].
bool bounds_of(const float (*coef)[3], int steps, Bounds& o)
{
	o.sx[0] = 1.0 + 1e-5;  // (the norm's rounding)
	for (int k = 0; k < steps; ++k)
	{
		const double a = coef[k][0], b = coef[k][1], c = coef[k][2], t = o.sx[k];
		if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
		o.sa[k] = t * t * (1.0 + 1e-5);
		auto h = [&](double l) { return fabs(a + l * (b + l * c)); };
		auto e = [&](double l) { return fabs(l * (b + l * c)); };
		o.sr[k] = e(o.sa[k]);
		double sp = std::max(h(0.0), h(o.sa[k]));  // of a + R
		const double turn = c != 0.0 ? -b / (2 * c) : -1.0;
		if (turn > 0.0 && turn < o.sa[k])
		{
			o.sr[k] = std::max(o.sr[k], e(turn));
			sp = std::max(sp, h(turn));
		}
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
		o.sx[k + 1] = most * (1.0 + 1e-4);
		if (!(o.sx[k + 1] <= 16.0) || !(o.sr[k] <= 256.0) || !(sp <= 256.0)) return false;
	}
	return true;
}

// 2^e with 2^e * bound < 2^15
float scale_under(double bound)
{
	int e = 0;
	frexp(bound, &e);  // bound < 2^e
	return ldexpf(1.0f, std::max(-40, std::min(15 - e, 40)));
}

// Returns X_0's scale.
float make_program(OrProgram& g, const float (*coef)[3], int steps)
{
	Bounds b;
	bounds_of(coef, steps, b);
	const float s0 = scale_under(b.sx[0]);
	float scale[ID_X + 2] = {0};  // of the matrices' present contents
	scale[ID_X] = s0;
	g.count = 0;
	// out = f A B + w E
	auto op = [&](int a, int bb, double f, int e, double w, int out, double bound) {
		OrOp& o = g.op[g.count++];
		o.a = (signed char)a; o.b = (signed char)bb; o.e = (signed char)e; o.out = (signed char)out;
		// (the scales are powers of two: the coefficients stay as they are)
		o.f = (float)(f / scale[a] / scale[bb]);
		o.w = e == ID_NONE ? 0.0f : (float)(w / scale[e]);
		o.so = out == ID_NONE ? 1.0f : scale_under(bound);
		if (out != ID_NONE) scale[out] = o.so;
	};
	for (int k = 0; k < steps; ++k)
	{
		const int x = ID_X + (k & 1), next = ID_X + (~k & 1);
		op(x, x, 1.0, ID_NONE, 0.0, ID_A, b.sa[k]);
		op(ID_A, ID_A, coef[k][2], ID_A, coef[k][1], ID_R, b.sr[k]);
		op(ID_R, x, 1.0, x, coef[k][0], k + 1 < steps ? next : ID_NONE, b.sx[k + 1]);
	}
	return s0;
}

// A launch's plan: the width of the tiles, how far they are split.
struct Plan
{
	int bn;
	int slots;  // of split tiles' parts
};

// About how many clocks (of 1.9 GHz), measured on rounds of one kind: an item of kb stages from its first copy to its last store,
// what a round costs beside its items (its barrier), and a round with split tiles on top (another barrier and the sums).  By these the faster width is
// taken within 5 % on twenty shapes from 130 x 400 to 2048 x 2048 (256 x 256 107 us by 64 columns, 169 by 128; 2048 x 2048 751 and 534).
long long item_clocks(int bn, long long kb) { return kb * (bn == 128 ? 900 : 550) + (bn == 128 ? 7000 : 5000); }
constexpr long long ROUND_CLOCKS = 3000, REDUCE_CLOCKS = 8000;

// Tiles of width bn: how far they are split, and about how many clocks the rounds take: for each the CTA with the most work.
long long plan_width(const OrParams& P, int bn, unsigned char (*split)[OR_MAX_OPS], unsigned long long* reduce, int* slots)
{
	long long total = 0;
	*reduce = 0;
	*slots = 0;
	for (int round = 0; round < P.prog.count; ++round)
	{
		const OrOp& o = P.prog.op[round];
		int tiles = 0;
		long long work = 0;
		auto each = [&](auto&& f) {
			for (int i = 0; i < P.count; ++i) f(i, op_tiles(o, P.mat[i].p, P.mat[i].q, bn), op_kb(o, P.mat[i].p, P.mat[i].q));
		};
		each([&](int, int n, int kb) {
			tiles += n;
			work += (long long)n * kb;
		});
		// whole tiles, or parts of about equal length for all matrices, so many that every SM has one
		const long long share = std::max<long long>(OR_SPLIT_K / OR_BK, (work + OR_SMS - 1) / OR_SMS);
		auto parts = [&](bool whole, int kb) { return whole ? 1 : (int)std::max<long long>(1, std::min<long long>(255, kb / share)); };
		auto clocks = [&](bool whole) {
			long long load[OR_SMS] = {0}, worst = 0;
			int t = 0, used = 0;
			each([&](int, int n, int kb) {
				const int s = parts(whole, kb);
				if (s > 1) used += n * s;
				const long long cost = item_clocks(bn, (kb + s - 1) / s);
				const long long rounds = (long long)n * s / OR_SMS;
				for (int c = 0; c < OR_SMS && rounds; ++c) load[c] += rounds * cost;
				const int rest = (int)((long long)n * s % OR_SMS);
				for (int c = 0; c < rest; ++c) load[(t + c) % OR_SMS] += cost;
				t = (t + rest) % OR_SMS;
			});
			for (long long l : load) worst = std::max(worst, l);
			return worst + ROUND_CLOCKS + (used ? REDUCE_CLOCKS : 0);
		};
		const long long cost = clocks(true);
		const long long cost_split = tiles * 2 <= OR_SMS ? clocks(false) : cost;
		const bool whole = cost <= cost_split;
		int used = 0;
		each([&](int i, int n, int kb) {
			split[i][round] = (unsigned char)parts(whole, kb);
			if (split[i][round] > 1) used += n * split[i][round];
		});
		if (used) *reduce |= 1ull << round;
		*slots = std::max(*slots, used);
		total += std::min(cost, cost_split);
	}
	return total;
}

size_t matrix_bytes(const OrMat& M)
{
	const size_t p = round_up((size_t)M.p, 128), q = round_up((size_t)M.q, 128);
	return (4 * p * q + 2 * OR_SQUARES * p * p) * sizeof(__half);
}

// Fills everything of P that does not depend on the workspace's address; returns the bytes of workspace.
size_t make_plan(OrParams& P, const OrthoArgs& a, const OrthoMatrix* m, int count, Plan& plan)
{
	memset(&P, 0, sizeof P);
	P.count = count;
	P.type = a.type;
	P.step = a.step;
	P.nesterov = a.nesterov;
	P.mu = a.mu;
	P.decay = a.decay;
	P.eps = a.eps;
	P.bad = a.bad;
	P.s0 = make_program(P.prog, a.coef, a.steps);
	for (int i = 0; i < count; ++i)
	{
		OrMat& M = P.mat[i];
		M.m = m[i];
		M.tall = M.m.rows > M.m.cols;
		M.p = std::min(M.m.rows, M.m.cols);
		M.q = std::max(M.m.rows, M.m.cols);
	}
	// the matrices with the longest products first: what is left for the last CTAs of a round is small
	std::stable_sort(P.mat, P.mat + count, [](const OrMat& x, const OrMat& y) { return (double)x.p * x.q > (double)y.p * y.q; });
	size_t bytes = 0;
	for (int i = 0; i < count; ++i)
	{
		OrMat& M = P.mat[i];
		M.ldx = (long long)round_up(M.q, 128);
		M.planex = M.ldx * (long long)round_up(M.p, 128);
		M.lds = (long long)round_up(M.p, 128);
		M.planes = M.lds * M.lds;
		M.units = P.units;
		M.units_per_row = (M.m.cols + OR_UNIT - 1) / OR_UNIT;
		P.units += M.units_per_row * ((M.m.rows + OR_UNIT - 1) / OR_UNIT);
		bytes += matrix_bytes(M);
	}
	long long best = -1;
	for (int bn : {128, 64})
	{
		static thread_local unsigned char split[ORTHO_MAX_MATRICES][OR_MAX_OPS];
		unsigned long long reduce;
		int slots;
		const long long c = plan_width(P, bn, split, &reduce, &slots);
		if (best >= 0 && c >= best) continue;
		best = c;
		plan.bn = bn;
		plan.slots = slots;
		P.reduce = reduce;
		memcpy(P.split, split, sizeof split);
	}
	return OR_HEADER + round_up(OR_SUMS, 256) + (size_t)plan.slots * 128 * plan.bn * sizeof(float) + bytes;
}

template <int BN>
bool make_maps(OrMaps& o, const OrMat& M)
{
	return tc_make_parts_map(&o.xa, M.X, M.p, M.q, M.ldx, M.planex, 4, OR_BK, TC_BM) &&
	       tc_make_parts_map(&o.xb, M.X, M.p, M.q, M.ldx, M.planex, 4, OR_BK, BN) &&
	       tc_make_parts_map_mn(&o.xn, M.X, M.p, M.q, M.ldx, M.planex, 4, OR_BK, BN) &&
	       tc_make_parts_map(&o.sa, M.S, M.p, M.p, M.lds, M.planes, 2 * OR_SQUARES, OR_BK, TC_BM) &&
	       tc_make_parts_map(&o.sb, M.S, M.p, M.p, M.lds, M.planes, 2 * OR_SQUARES, OR_BK, BN);
}

template <int BN>
cudaError_t launch_width(OrParams& P, cudaStream_t s)
{
	for (int i = 0; i < P.count; ++i)
		if (!make_maps<BN>(P.maps[i], P.mat[i])) return cudaErrorInvalidValue;
	int sms = 0;
	cudaError_t e = prepare_tc_launch(reinterpret_cast<const void*>(ortho_kernel<BN>), OrSmem<BN>::TOTAL, &sms);
	if (e != cudaSuccess) return e;
	// no more CTAs than the largest round has items and pieces
	int most = P.units;
	for (int round = 0; round < P.prog.count; ++round)
	{
		int n = 0, splits = 0;
		for (int i = 0; i < P.count; ++i)
		{
			const int tiles = op_tiles(P.prog.op[round], P.mat[i].p, P.mat[i].q, BN);
			n += tiles * P.split[i][round];
			if (P.split[i][round] > 1) splits += tiles;
		}
		P.items[round] = n;
		P.splits[round] = splits;
		most = std::max(most, std::max(n, splits * OrSmem<BN>::PIECES));
	}
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned)std::min(std::min(sms, OR_SMS), most));
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

thread_local OrParams t_params;

}  // namespace

bool ortho_coefficients_ok(const float (*coef)[3], int steps)
{
	Bounds b;
	return bounds_of(coef, steps, b);
}

// (whatever the steps, the coefficients and the plan that they lead to)
size_t ortho_workspace_bytes(const OrthoMatrix* m, int count)
{
	size_t most = 0;
	for (int first = 0; first < count; first += ORTHO_MAX_MATRICES)
	{
		size_t bytes = 0;
		double parts = 0.0;  // of split tiles, at most one per SM
		for (int i = first; i < std::min(count, first + ORTHO_MAX_MATRICES); ++i)
		{
			OrMat M;
			M.p = std::min(m[i].rows, m[i].cols);
			M.q = std::max(m[i].rows, m[i].cols);
			bytes += matrix_bytes(M);
			if (M.q > OR_SPLIT_K) parts += ceil(M.p / 128.0) * ceil(M.q / 64.0) * ceil(M.q / (double)OR_SPLIT_K);
		}
		most = std::max(most, bytes + (size_t)std::min(parts, (double)OR_SMS) * 128 * 128 * sizeof(float));
	}
	return 256 + OR_HEADER + round_up(OR_SUMS, 256) + most;  // (256: the caller's pointer need not be aligned)
}

int* ortho_status(void* work) { return reinterpret_cast<int*>(round_up((size_t)work, 256)); }

cudaError_t launch_orthogonalize(const OrthoArgs& a, void* work, size_t work_bytes, cudaStream_t s)
{
	OrParams& P = t_params;
	for (int first = 0; first < a.count; first += ORTHO_MAX_MATRICES)
	{
		// A list of small matrices only goes to one CTA for each of them; beside larger ones they ride along, but single rows and
		// columns, which go to one CTA each behind the others.
		const int all = std::min(ORTHO_MAX_MATRICES, a.count - first);
		int* const status = a.status ? a.status : ortho_status(work);
		const bool reset = first == 0 && !a.status;
		OrthoMatrix m[ORTHO_MAX_MATRICES], vectors[ORTHO_MAX_MATRICES];
		int count = 0, n = 0;
		bool small = true;
		for (int i = first; i < first + all; ++i)
		{
			const OrthoMatrix& x = a.mat[i];
			if (ortho_vector(x)) vectors[n++] = x;
			else
			{
				small = small && ortho_small(x.rows, x.cols);
				m[count++] = x;
			}
		}
		if (small)
			while (n > 0) m[count++] = vectors[--n];
		if (small)
		{
			const float s0 = make_program(P.prog, a.coef, a.steps);
			const cudaError_t e = launch_ortho_small(a, P.prog, s0, m, count, status, reset, false, s);
			if (e != cudaSuccess) return e;
			continue;
		}
		Plan plan;
		const size_t need = make_plan(P, a, m, count, plan);
		if (need + 256 > work_bytes) return cudaErrorInvalidValue;
		char* at = reinterpret_cast<char*>(ortho_status(work));
		P.status = status;
		P.reset = reset;
		at += OR_HEADER;
		P.arrived = reinterpret_cast<unsigned*>(at - OR_HEADER / 2);
		P.sums = reinterpret_cast<double*>(at);
		at += round_up(OR_SUMS, 256);
		P.part = reinterpret_cast<float4*>(at);
		at += (size_t)plan.slots * 128 * plan.bn * sizeof(float);
		for (int i = 0; i < P.count; ++i)
		{
			OrMat& M = P.mat[i];
			M.X = reinterpret_cast<__half*>(at);
			M.S = M.X + 4 * M.planex;
			at += matrix_bytes(M);
		}
		cudaError_t e = plan.bn == 128 ? launch_width<128>(P, s) : launch_width<64>(P, s);
		if (e == cudaSuccess && n > 0) e = launch_ortho_small(a, P.prog, P.s0, vectors, n, status, false, true, s);
		if (e != cudaSuccess) return e;
	}
	return cudaSuccess;
}

}  // namespace glb
