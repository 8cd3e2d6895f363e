// extern "C" layer of the operators on device buffers (declared in include/glades_b200.h): their arguments are checked here,
// their work is queued on the caller's stream.  Nothing is allocated, nothing waits, no state is kept between calls.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <new>
#include <utility>
#include <vector>

#include "internal.h"
#include "orthogonalize.h"

using namespace glb;

namespace {

// The call's device made current, the caller's put back.
struct OnDevice
{
	int before = -1;
	cudaError_t error;
	explicit OnDevice(int device)
	{
		error = cudaGetDevice(&before);
		if (error == cudaSuccess && before != device) error = cudaSetDevice(device);
		if (error == cudaSuccess && before == device) before = -1;
	}
	~OnDevice()
	{
		if (before >= 0) cudaSetDevice(before);
	}
};

// GL_OK for an sm_100 device; its attributes are asked for once
int check_device(int device)
{
	static std::atomic<int> known[64];  // 1: sm_100
	if (device < 0 || device >= 64) return report_error(GL_ERR_INVALID, "device %d: no such device", device);
	if (known[device] == 1) return GL_OK;
	int n = 0, major = 0;
	if (cudaGetDeviceCount(&n) != cudaSuccess || n < 1)
	{
		cudaGetLastError();
		return report_error(GL_ERR_NO_DEVICE, "no sm_100 CUDA device");
	}
	if (device >= n) return report_error(GL_ERR_INVALID, "device %d: no such device", device);
	if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device) != cudaSuccess || major != 10)
	{
		cudaGetLastError();
		return report_error(GL_ERR_NO_DEVICE, "device %d is not an sm_100 device", device);
	}
	known[device] = 1;
	return GL_OK;
}

int type_size(int type) { return type == GL_F32 ? 4 : 2; }
bool type_ok(int type) { return type == GL_F32 || type == GL_BF16 || type == GL_F16; }
bool on(const void* p, int bytes) { return (uintptr_t)p % bytes == 0; }

constexpr long long MAX_DIM = 1ll << 30;     // rows or columns of a matrix
constexpr long long MAX_PITCH = 1ll << 40;

// a [rows][cols] matrix of elements of `size` bytes
bool matrix_ok(const void* p, long long ld, long long cols, int size) { return p && on(p, size) && ld >= cols && ld <= MAX_PITCH; }

int finish(const char* name, cudaError_t e)
{
	if (e == cudaSuccess) return GL_OK;
	return report_error(GL_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

int check_steps(const char* name, OrthoArgs& a, const float* coefficients, int steps, float eps, int type)
{
	if (steps < 1 || steps > ORTHO_MAX_STEPS) return report_error(GL_ERR_INVALID, "%s: steps must be 1 to %d", name, ORTHO_MAX_STEPS);
	if (!type_ok(type)) return report_error(GL_ERR_INVALID, "%s: unknown element type %d", name, type);
	if (!(eps >= 0.0f) || isinf(eps)) return report_error(GL_ERR_INVALID, "%s: eps must be a number >= 0", name);
	for (int k = 0; k < steps; ++k)
		for (int j = 0; j < 3; ++j) a.coef[k][j] = coefficients ? coefficients[3 * k + j] : ORTHO_QUINTIC[j];
	if (!ortho_coefficients_ok(a.coef, steps))
		return report_error(GL_ERR_INVALID, "%s: under these coefficients a singular value could grow beyond 16", name);
	a.steps = steps;
	a.eps = eps;
	a.type = type;
	a.status = nullptr;
	return GL_OK;
}

bool shape_ok(int rows, int cols) { return rows >= 1 && cols >= 1 && rows <= MAX_DIM && cols <= MAX_DIM; }

// The arguments of a list of matrices, each input with the number of the output that may take its place (-1: none may).
struct Arguments
{
	std::vector<std::pair<uintptr_t, int>> in, out;
	void read(const void* p, int output) { in.push_back({(uintptr_t)p, output}); }
	void write(const void* p, int output) { out.push_back({(uintptr_t)p, output}); }
	// No output begins where another one does, or where an input of another one's does: the matrices are worked on at once.
	bool apart()
	{
		std::sort(out.begin(), out.end());
		for (size_t i = 1; i < out.size(); ++i)
			if (out[i].first == out[i - 1].first) return false;
		for (const auto& a : in)
		{
			const auto o = std::lower_bound(out.begin(), out.end(), std::make_pair(a.first, -1));
			if (o != out.end() && o->first == a.first && o->second != a.second) return false;
		}
		return true;
	}
};

template <class ITEM>
int64_t workspace(const char* name, const ITEM* items, int count)
{
	if (count < 0 || (count > 0 && !items)) return report_error(GL_ERR_INVALID, "%s: bad argument", name);
	try
	{
		std::vector<OrthoMatrix> m(count);
		double total = 0.0;
		for (int i = 0; i < count; ++i)
		{
			if (!shape_ok(items[i].rows, items[i].cols)) return report_error(GL_ERR_INVALID, "%s: matrix %d has no rows or no columns", name, i);
			m[i].rows = items[i].rows;
			m[i].cols = items[i].cols;
			total += 64.0 * ((double)items[i].rows + 128) * ((double)items[i].cols + 128);
		}
		if (total > 4e18) return report_error(GL_ERR_TOO_LARGE, "%s: the matrices are too large", name);
		return (int64_t)ortho_workspace_bytes(m.data(), count);
	}
	catch (const std::bad_alloc&)
	{
		return report_error(GL_ERR_INVALID, "%s: no host memory for %d matrices", name, count);
	}
}

int run_ortho(const char* name, OrthoArgs& a, const std::vector<OrthoMatrix>& m, void* d_work, int64_t work_bytes, void* stream, int device)
{
	a.mat = m.data();
	a.count = (int)m.size();
	if (a.count == 0 && (!d_work || work_bytes < (int64_t)ortho_workspace_bytes(nullptr, 0))) return GL_OK;
	if (!d_work || work_bytes < (int64_t)ortho_workspace_bytes(a.mat, a.count))
		return report_error(GL_ERR_INVALID, "%s: the workspace is too small", name);
	if (int r = check_device(device)) return r;
	OnDevice guard(device);
	if (guard.error != cudaSuccess) return finish(name, guard.error);
	// (a workspace needs no initialisation: its status is this call's, whatever it held)
	if (a.count == 0) return finish(name, cudaMemsetAsync(ortho_status(d_work), 0, sizeof(int), static_cast<cudaStream_t>(stream)));
	return finish(name, launch_orthogonalize(a, d_work, (size_t)work_bytes, static_cast<cudaStream_t>(stream)));
}

}  // namespace

extern "C" int gl_layer_norm(const void* d_x, int64_t ldx, const float* d_gain, const float* d_shift, void* d_y, int64_t ldy, float* d_mean,
                             float* d_rstd, int64_t rows, int32_t n, float eps, int32_t type, void* stream, int32_t device)
{
	if (!type_ok(type)) return report_error(GL_ERR_INVALID, "gl_layer_norm: unknown element type %d", type);
	if (rows < 0 || n < 1 || n > MAX_DIM || !(eps >= 0.0f) || isinf(eps)) return report_error(GL_ERR_INVALID, "gl_layer_norm: bad size or eps");
	if (rows == 0) return GL_OK;
	const int size = type_size(type);
	if (!matrix_ok(d_x, ldx, n, size) || !matrix_ok(d_y, ldy, n, size))
		return report_error(GL_ERR_INVALID, "gl_layer_norm: x or y is missing, off its type's boundary, or its pitch is below n");
	if (!on(d_gain, 4) || !on(d_shift, 4) || !on(d_mean, 4) || !on(d_rstd, 4))
		return report_error(GL_ERR_INVALID, "gl_layer_norm: an fp32 vector lies off a 4-byte boundary");
	if (d_y == d_x && ldx != ldy) return report_error(GL_ERR_INVALID, "gl_layer_norm: in place needs one pitch");
	if (int r = check_device(device)) return r;
	OnDevice guard(device);
	if (guard.error != cudaSuccess) return finish("gl_layer_norm", guard.error);
	LayerNormArgs a = {};
	a.x = d_x; a.ldx = ldx;
	a.y = d_y; a.ldy = ldy;
	a.gain = d_gain; a.shift = d_shift;
	a.mean = d_mean; a.rstd = d_rstd;
	a.rows = rows; a.n = n; a.eps = eps;
	return finish("gl_layer_norm", launch_layer_norm(a, type, static_cast<cudaStream_t>(stream)));
}

extern "C" int64_t gl_layer_norm_backward_workspace(int64_t rows, int32_t n)
{
	if (rows < 0 || n < 1 || n > MAX_DIM) return report_error(GL_ERR_INVALID, "gl_layer_norm_backward_workspace: bad size");
	return (int64_t)(layer_norm_partial_rows(rows, n) * (size_t)n * sizeof(float2) + 15);
}

extern "C" int gl_layer_norm_backward(const void* d_dy, int64_t lddy, const void* d_x, int64_t ldx, const float* d_gain, const float* d_mean,
                                      const float* d_rstd, void* d_dx, int64_t lddx, float* d_dgain, float* d_dshift, int64_t rows, int32_t n,
                                      int32_t type, void* d_work, int64_t work_bytes, void* stream, int32_t device)
{
	const char* name = "gl_layer_norm_backward";
	if (!type_ok(type)) return report_error(GL_ERR_INVALID, "%s: unknown element type %d", name, type);
	if (rows < 0 || n < 1 || n > MAX_DIM) return report_error(GL_ERR_INVALID, "%s: bad size", name);
	const int size = type_size(type);
	if (!on(d_gain, 4) || !on(d_mean, 4) || !on(d_rstd, 4) || !on(d_dgain, 4) || !on(d_dshift, 4))
		return report_error(GL_ERR_INVALID, "%s: an fp32 vector lies off a 4-byte boundary", name);
	const bool sums = d_dgain || d_dshift;
	if (rows > 0)
	{
		if (!matrix_ok(d_dy, lddy, n, size) || !matrix_ok(d_x, ldx, n, size) || (d_dx && !matrix_ok(d_dx, lddx, n, size)))
			return report_error(GL_ERR_INVALID, "%s: a matrix is missing, off its type's boundary, or its pitch is below n", name);
		if (!d_mean || !d_rstd) return report_error(GL_ERR_INVALID, "%s: the forward pass's mean and rstd are needed", name);
		if ((d_dx == d_x && d_dx && lddx != ldx) || (d_dx == d_dy && d_dx && lddx != lddy))
			return report_error(GL_ERR_INVALID, "%s: in place needs one pitch", name);
		if (sums && (!d_work || work_bytes < gl_layer_norm_backward_workspace(rows, n)))
			return report_error(GL_ERR_INVALID, "%s: the workspace is too small", name);
	}
	if (int r = check_device(device)) return r;
	OnDevice guard(device);
	if (guard.error != cudaSuccess) return finish(name, guard.error);
	const cudaStream_t s = static_cast<cudaStream_t>(stream);
	if (rows == 0)
	{
		cudaError_t e = d_dgain ? cudaMemsetAsync(d_dgain, 0, (size_t)n * sizeof(float), s) : cudaSuccess;
		if (e == cudaSuccess && d_dshift) e = cudaMemsetAsync(d_dshift, 0, (size_t)n * sizeof(float), s);
		return finish(name, e);
	}
	if (!d_dx && !sums) return GL_OK;
	LayerNormArgs a = {};
	a.x = d_x; a.ldx = ldx;
	a.dy = d_dy; a.lddy = lddy;
	a.dx = d_dx; a.lddx = lddx;
	a.gain = d_gain;
	a.mean = const_cast<float*>(d_mean);
	a.rstd = const_cast<float*>(d_rstd);
	a.part = sums ? reinterpret_cast<float2*>(((uintptr_t)d_work + 15) / 16 * 16) : nullptr;
	a.dgain = d_dgain; a.dshift = d_dshift;
	a.rows = rows; a.n = n;
	return finish(name, launch_layer_norm_backward(a, type, s));
}

extern "C" int64_t gl_orthogonalize_workspace(const gl_ortho_item* items, int32_t count)
{
	return workspace("gl_orthogonalize_workspace", items, count);
}

extern "C" int64_t gl_muon_workspace(const gl_muon_item* items, int32_t count) { return workspace("gl_muon_workspace", items, count); }

extern "C" int gl_orthogonalize(const gl_ortho_item* items, int32_t count, const float* coefficients, int32_t steps, float eps, int32_t type,
                                void* d_work, int64_t work_bytes, void* stream, int32_t device)
{
	const char* name = "gl_orthogonalize";
	if (count < 0 || (count > 0 && !items)) return report_error(GL_ERR_INVALID, "%s: bad argument", name);
	OrthoArgs a = {};
	if (int r = check_steps(name, a, coefficients, steps, eps, type)) return r;
	const int size = type_size(type);
	try
	{
		std::vector<OrthoMatrix> m(count);
		Arguments all;
		for (int i = 0; i < count; ++i)
		{
			const gl_ortho_item& t = items[i];
			if (!shape_ok(t.rows, t.cols)) return report_error(GL_ERR_INVALID, "%s: matrix %d has no rows or no columns", name, i);
			if (!matrix_ok(t.d_in, t.ld_in, t.cols, size) || !matrix_ok(t.d_out, t.ld_out, t.cols, size))
				return report_error(GL_ERR_INVALID, "%s: matrix %d is missing, off its type's boundary, or its pitch is below its columns", name, i);
			m[i].rows = t.rows; m[i].cols = t.cols;
			m[i].grad = t.d_in; m[i].ld_grad = t.ld_in;
			m[i].out = t.d_out; m[i].ld_out = t.ld_out;
			all.read(t.d_in, i);
			all.write(t.d_out, i);
		}
		if (!all.apart()) return report_error(GL_ERR_INVALID, "%s: an output is listed twice, or is another matrix's input", name);
		return run_ortho(name, a, m, d_work, work_bytes, stream, device);
	}
	catch (const std::bad_alloc&)
	{
		return report_error(GL_ERR_INVALID, "%s: no host memory for %d matrices", name, count);
	}
}

extern "C" int gl_muon_step(const gl_muon_item* items, int32_t count, float momentum, int32_t nesterov, float weight_decay,
                            const float* coefficients, int32_t steps, float eps, int32_t type, void* d_work, int64_t work_bytes, void* stream,
                            int32_t device)
{
	const char* name = "gl_muon_step";
	if (count < 0 || (count > 0 && !items)) return report_error(GL_ERR_INVALID, "%s: bad argument", name);
	if (!isfinite(momentum) || !isfinite(weight_decay)) return report_error(GL_ERR_INVALID, "%s: momentum and weight decay must be numbers", name);
	OrthoArgs a = {};
	if (int r = check_steps(name, a, coefficients, steps, eps, type)) return r;
	a.step = 1;
	a.nesterov = nesterov != 0;
	a.mu = momentum;
	a.decay = weight_decay;
	const int size = type_size(type);
	try
	{
		std::vector<OrthoMatrix> m(count);
		Arguments all;
		for (int i = 0; i < count; ++i)
		{
			const gl_muon_item& t = items[i];
			if (!shape_ok(t.rows, t.cols)) return report_error(GL_ERR_INVALID, "%s: matrix %d has no rows or no columns", name, i);
			if (!matrix_ok(t.d_grad, t.ld_grad, t.cols, size) || !matrix_ok(t.d_momentum, t.ld_momentum, t.cols, 4) ||
			    !matrix_ok(t.d_momentum_out, t.ld_momentum, t.cols, 4) || !matrix_ok(t.d_weight, t.ld_weight, t.cols, 4) ||
			    !matrix_ok(t.d_weight_out, t.ld_weight, t.cols, 4))
				return report_error(GL_ERR_INVALID, "%s: matrix %d is missing, off its type's boundary, or its pitch is below its columns", name, i);
			if (!isfinite(t.lr)) return report_error(GL_ERR_INVALID, "%s: the learning rate of matrix %d is no number", name, i);
			m[i].rows = t.rows; m[i].cols = t.cols;
			m[i].grad = t.d_grad; m[i].ld_grad = t.ld_grad;
			m[i].mom = t.d_momentum; m[i].mom_out = t.d_momentum_out; m[i].ld_mom = t.ld_momentum;
			m[i].w = t.d_weight; m[i].w_out = t.d_weight_out; m[i].ld_w = t.ld_weight;
			m[i].lr = t.lr;
			all.read(t.d_grad, -1);
			all.read(t.d_momentum, 2 * i);
			all.read(t.d_weight, 2 * i + 1);
			all.write(t.d_momentum_out, 2 * i);
			all.write(t.d_weight_out, 2 * i + 1);
		}
		if (!all.apart()) return report_error(GL_ERR_INVALID, "%s: an output is listed twice, or is another argument than its own input", name);
		return run_ortho(name, a, m, d_work, work_bytes, stream, device);
	}
	catch (const std::bad_alloc&)
	{
		return report_error(GL_ERR_INVALID, "%s: no host memory for %d matrices", name, count);
	}
}

extern "C" int gl_orthogonalize_status(const void* d_work, void* stream, int32_t device)
{
	const char* name = "gl_orthogonalize_status";
	if (!d_work) return report_error(GL_ERR_INVALID, "%s: no workspace", name);
	if (int r = check_device(device)) return r;
	OnDevice guard(device);
	if (guard.error != cudaSuccess) return finish(name, guard.error);
	int code = 0;
	const cudaStream_t s = static_cast<cudaStream_t>(stream);
	cudaError_t e = cudaMemcpyAsync(&code, ortho_status(const_cast<void*>(d_work)), sizeof code, cudaMemcpyDeviceToHost, s);
	if (e == cudaSuccess) e = cudaStreamSynchronize(s);
	if (e != cudaSuccess) return finish(name, e);
	if (code) return report_error(GL_ERR_TIMEOUT, "%s: a bounded wait inside the orthogonalisation ran out (role %d)", name, code);
	return GL_OK;
}
