#include "ops_inst.cuh"

namespace b200 {

const OpKernels kOpKernelsF16 = OpInstances<kOpF16>::kTable;

} // namespace b200
