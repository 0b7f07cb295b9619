// ops_residual_norm_vec.cu -- the residual norm's backward for rows that move as float4: eight columns per
// thread (16 above 8192), up to 256, 512 or 1024 threads to a row.
#include "nnb_residual_norm.cuh"

namespace nnb {
namespace resnorm {

nnb_status residual_norm_bwd_vec(cudaStream_t s, const Grad& p, long long groups) {
	if (p.D > 8 * 1024) return launch_bwd<4, 4, 1024>(s, p, groups);
	if (p.T > 512) return launch_bwd<4, 2, 1024>(s, p, groups);
	if (p.T > kCta) return launch_bwd<4, 2, 512>(s, p, groups);
	return launch_bwd<4, 2, kCta>(s, p, groups);
}

}  // namespace resnorm
}  // namespace nnb
