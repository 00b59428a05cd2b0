#include "ops_inst.cuh"

namespace b200 {

const OpKernels kOpKernelsTF32 = OpInstances<kOpTF32>::kTable;

} // namespace b200
