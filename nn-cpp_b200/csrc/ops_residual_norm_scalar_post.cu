// ops_residual_norm_scalar_post.cu -- instances of the residual norm's backward: rows of any length and alignment, moved as single floats,
// with a norm after the block.
#include "nnb_residual_norm.cuh"

namespace nnb {
namespace resnorm {

nnb_status bwd_scalar_post(cudaStream_t s, const Grad& p, long long groups) {
	if (p.layer)
		return p.gate ? dispatch_bwd<1, true, true, true>(s, p, groups) : dispatch_bwd<1, true, true, false>(s, p, groups);
	return p.gate ? dispatch_bwd<1, false, true, true>(s, p, groups) : dispatch_bwd<1, false, true, false>(s, p, groups);
}

}  // namespace resnorm
}  // namespace nnb
