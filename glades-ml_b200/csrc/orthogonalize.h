// Orthogonalisation of matrices and the weight update built on it (orthogonalize.cu).
#pragma once
#include "internal.h"

namespace glb {

constexpr int ORTHO_MAX_MATRICES = GL_MAX_WEIGHT_LAYERS;  // of one launch
constexpr int ORTHO_MAX_STEPS = 16;
constexpr float ORTHO_QUINTIC[3] = {3.4445f, -4.7750f, 2.0315f};  // the usual coefficients
constexpr float ORTHO_EPS = 1e-7f;

// One row-major matrix.  Orthogonalisation: out = O(grad).  Update step: mom_out = mu mom + grad,
// w_out = (1 - lr decay) w - lr O(u) with u = grad + mu mom_out (nesterov) or mom_out.
struct OrthoMatrix
{
	int rows, cols;
	const void* grad;
	long long ld_grad;
	void* out;
	long long ld_out;
	const float* mom;
	float* mom_out;
	long long ld_mom;
	const float* w;
	float* w_out;
	long long ld_w;
	float lr;
};
struct OrthoArgs
{
	const OrthoMatrix* mat;
	int count, steps, type, step, nesterov;
	float mu, decay, eps;
	float coef[ORTHO_MAX_STEPS][3];
	int* bad;     // device word whose bit 0 a new weight that is not finite sets, or NULL
	int* status;  // device word that a wait that runs out raises, or NULL: the workspace's
};
// false where the coefficients let a singular value of [0, 1] (or an eigenvalue on the way) leave the range that the parts are
// scaled for
bool ortho_coefficients_ok(const float (*coef)[3], int steps);
size_t ortho_workspace_bytes(const OrthoMatrix* m, int count);  // (only the shapes are looked at)
int* ortho_status(void* work);  // where a workspace keeps its status word
cudaError_t launch_orthogonalize(const OrthoArgs& a, void* work, size_t work_bytes, cudaStream_t s);

}  // namespace glb
