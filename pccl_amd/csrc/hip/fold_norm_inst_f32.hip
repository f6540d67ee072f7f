// fold_norm_inst_f32.hip -- instantiates the norms around a block for f32 rows and parameters.
#include "fold_norm_kernel.h"

namespace pccl_dev {
PCCL_DEFINE_FOLD_NORM(PCCL_F32, true)
}  // namespace pccl_dev
