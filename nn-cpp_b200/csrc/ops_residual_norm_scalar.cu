// ops_residual_norm_scalar.cu -- the residual norm's backward for rows of any length and alignment, as the
// float4 form with single floats.
#include "nnb_residual_norm.cuh"

namespace nnb {
namespace resnorm {

nnb_status residual_norm_bwd_scalar(cudaStream_t s, const Grad& p, long long groups) {
	if (p.D > 8 * 1024) return launch_bwd<1, 16, 1024>(s, p, groups);
	if (p.T > 512) return launch_bwd<1, 8, 1024>(s, p, groups);
	if (p.T > kCta) return launch_bwd<1, 8, 512>(s, p, groups);
	return launch_bwd<1, 8, kCta>(s, p, groups);
}

}  // namespace resnorm
}  // namespace nnb
