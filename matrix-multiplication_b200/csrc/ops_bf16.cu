#include "ops_inst.cuh"

namespace b200 {

const OpKernels kOpKernelsBF16 = OpInstances<kOpBF16>::kTable;

} // namespace b200
