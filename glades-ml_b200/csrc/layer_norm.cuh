// What the layer norm's kernels share (layer_norm.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "internal.h"

namespace glb {

constexpr int LN_SMS = 148;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b)
{
	f32x2 r;
	asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
	return r;
}
// a word of two 16-bit values as floats, and back
template <class T> __device__ __forceinline__ f32x2 word_pair(unsigned w);
template <> __device__ __forceinline__ f32x2 word_pair<__nv_bfloat16>(unsigned w) { return pair2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
template <> __device__ __forceinline__ f32x2 word_pair<__half>(unsigned w)
{
	const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
	return pair2(f.x, f.y);
}
template <class T> __device__ __forceinline__ unsigned pair_word(f32x2 v);
template <> __device__ __forceinline__ unsigned pair_word<__nv_bfloat16>(f32x2 v)
{
	float lo, hi;
	unpair2(v, lo, hi);
	const __nv_bfloat162 w = __floats2bfloat162_rn(lo, hi);
	return *reinterpret_cast<const unsigned*>(&w);
}
template <> __device__ __forceinline__ unsigned pair_word<__half>(f32x2 v)
{
	float lo, hi;
	unpair2(v, lo, hi);
	const __half2 w = __floats2half2_rn(lo, hi);
	return *reinterpret_cast<const unsigned*>(&w);
}

// 1 / sqrt(v): the fast root, and a Newton step that brings it to within 2 units in the last place (a division and a root are 60
// instructions of every lane of a row)
__device__ __forceinline__ float inverse_root(float v)
{
	const float r = rsqrtf(v);
	const float e = fmaf(-v * r, r, 1.0f);
	return v > 1e-37f && v < 3.0e38f ? fmaf(0.5f * r, e, r) : 1.0f / sqrtf(v);
}

// 16 bytes from global to shared memory, or zeros; not waited for.
__device__ __forceinline__ void copy_ahead(void* to, const void* from, bool copy)
{
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from), "r"(copy ? 16 : 0) : "memory");
}

// A lane's access to a row, kept as it came: 16 bytes, or two values.
template <class T, int VEC>
struct Pack
{
	static constexpr int WORDS = VEC * (int)sizeof(T) / 4;
	unsigned w[WORDS];
	__device__ __forceinline__ void load(const T* p)
	{
		if constexpr (WORDS == 1) w[0] = *reinterpret_cast<const unsigned*>(p);
		else if constexpr (WORDS == 4)
		{
			const uint4 v = *reinterpret_cast<const uint4*>(p);
			w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
		}
	}
	__device__ __forceinline__ void store(T* p) const
	{
		if constexpr (WORDS == 1) *reinterpret_cast<unsigned*>(p) = w[0];
		else if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
	}
	__device__ __forceinline__ void put(int h, T v)
	{
		if constexpr (sizeof(T) == 2) w[0] |= (unsigned)*reinterpret_cast<const unsigned short*>(&v) << (16 * h);
		else w[h] = *reinterpret_cast<const unsigned*>(&v);
	}
	__device__ __forceinline__ void set(uint4 v) { w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
	__device__ __forceinline__ f32x2 pair(int i) const
	{
		if constexpr (sizeof(T) == 2) return word_pair<T>(w[i]);
		else return pair2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
	}
	__device__ __forceinline__ void set_pair(int i, f32x2 v)
	{
		if constexpr (sizeof(T) == 2) w[i] = pair_word<T>(v);
		else
		{
			float lo, hi;
			unpair2(v, lo, hi);
			w[2 * i] = __float_as_uint(lo);
			w[2 * i + 1] = __float_as_uint(hi);
		}
	}
	__device__ __forceinline__ void clear()
	{
#pragma unroll
		for (int i = 0; i < WORDS; ++i) w[i] = 0;
	}
};

}  // namespace glb
