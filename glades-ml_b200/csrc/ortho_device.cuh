// What the kernels of the orthogonalisation share: programs of products, the caller's elements, parts, waits and MMAs of a
// warp that stays together (orthogonalize.cu, ortho_small.cu).
#pragma once
#include <algorithm>

#include <cuda_bf16.h>

#include "ortho_walk.h"
#include "orthogonalize.h"
#include "tc_device.cuh"

namespace glb {
using namespace tc;

// Three products a step, one behind the other: A = X X^T, R = b A + c A A, X <- a X + R X.
constexpr int OR_MAX_OPS = 3 * ORTHO_MAX_STEPS;

struct OrProgram
{
	OrOp op[OR_MAX_OPS];
	int count;
};

// What X_0 is U times, from the sum of U's squares: in 64 bits throughout, since finite elements may have a norm beyond fp32's range.
// A zero matrix without an eps stays zero.
__device__ __forceinline__ double inverse_norm(double sum, float eps)
{
	const double norm = sqrt(sum) + (double)eps;
	return norm == 0.0 ? 0.0 : 1.0 / norm;
}

// ---- elements of the caller's matrices, four neighbours at a time ------------------------------------------------
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
// `left` of them exist; wide: a 16-byte (8-byte) boundary
__device__ __forceinline__ void load4(const void* p, long long i, int type, bool wide, int left, float (&v)[4])
{
	if (wide && left >= 4)
	{
		if (type == GL_F32)
		{
			const float4 w = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
			v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
			return;
		}
		const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(p) + i);
#pragma unroll
		for (int k = 0; k < 4; ++k)
		{
			const unsigned short u = (unsigned short)((k < 2 ? w.x : w.y) >> (16 * (k & 1)));
			v[k] = type == GL_BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
		}
		return;
	}
#pragma unroll
	for (int k = 0; k < 4; ++k) v[k] = k < left ? load_typed(p, i + k, type) : 0.0f;
}
__device__ __forceinline__ void store4(float* p, long long i, bool wide, int left, const float (&v)[4])
{
	if (wide && left >= 4)
	{
		*reinterpret_cast<float4*>(p + i) = make_float4(v[0], v[1], v[2], v[3]);
		return;
	}
#pragma unroll
	for (int k = 0; k < 4; ++k)
		if (k < left) p[i + k] = v[k];
}

// hi and lo of x * s, lo unscaled
__device__ __forceinline__ void split_pair(float x, float y, float s, uint32_t& hi, uint32_t& lo)
{
	const float xs = x * s, ys = y * s;
	const __half2 h = __floats2half2_rn(xs, ys);
	const float2 f = __half22float2(h);
	const __half2 l = __floats2half2_rn(xs - f.x, ys - f.y);
	hi = *reinterpret_cast<const uint32_t*>(&h);
	lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ bool elect_one()
{
	uint32_t p;
	asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
	return p != 0;
}
// A bounded wait of a whole warp, which stays together: what the issuing warps compute can then live in uniform registers
// (one lane on its own spends 70 clocks on the operands of every MMA it issues).
__device__ __noinline__ static bool warp_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err_flag, int code)
{
	const long long t0 = clock64();
	for (;;)
	{
		if (__all_sync(0xFFFFFFFFu, mbar_try(bar, parity))) return true;
		if (__any_sync(0xFFFFFFFFu, *abort_flag != 0)) return false;
		if (__any_sync(0xFFFFFFFFu, clock64() - t0 > TC_WAIT_CYCLES))
		{
			if ((threadIdx.x & 31) == 0)
			{
				*abort_flag = 1;
				atomicExch(err_flag, code);
			}
			return false;
		}
	}
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err_flag, int code)
{
	return __all_sync(0xFFFFFFFFu, mbar_try(bar, parity)) || warp_wait_slow(bar, parity, abort_flag, err_flag, code);
}
// tcgen05.mma with descriptors given as a low word (the address moves) and a high word that stays; the accumulator is added to,
// or (first) replaced
__device__ __forceinline__ void mma(bool first, uint32_t d, uint32_t a, uint32_t a_high, uint32_t b, uint32_t b_high, uint32_t idesc)
{
	asm volatile(
	    "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
	    "mov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
	    "setp.eq.u32 p, %6, 0;\n\t"
	    "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d),
	    "r"(a), "r"(a_high), "r"(b), "r"(b_high), "r"(idesc), "r"((uint32_t)first)
	    : "memory");
}

// small matrices (ortho_small.cu): whether one is, whether one is a single row or column, and the launch for m[0] .. [count - 1], each of
// which is one or the other (beside: single rows and columns only, which may run beside the kernel in front of them on the stream)
bool ortho_small(int rows, int cols);
bool ortho_vector(const OrthoMatrix& m);
cudaError_t launch_ortho_small(const OrthoArgs& a, const OrProgram& prog, float s0, const OrthoMatrix* m, int count, int* status, bool reset, bool beside, cudaStream_t s);

}  // namespace glb
