// The kernels of linear maps (nd_linear.hpp) for float16.
#include "nd_linear_types.hpp"

namespace nd {
template hipError_t launch_linear<_Float16>(const LinearParams&, Layout, After, const LinearPlan&, hipStream_t);
template hipError_t launch_pair<_Float16>(const LinearParams&, After, const LinearPlan&, const LinearParams&, const LinearPlan&, hipStream_t);
template hipError_t launch_again<_Float16>(const LinearParams&, const LinearPlan&, hipStream_t);
template hipError_t launch_joins<_Float16>(const Joins&, uint32_t, hipStream_t);
template hipError_t launch_few_rows<_Float16>(const LinearParams&, After, hipStream_t);
template hipError_t launch_slope<_Float16>(const LinearParams&, const void*, int64_t, float*, void*, int64_t, float*, hipStream_t);
}  // namespace nd
