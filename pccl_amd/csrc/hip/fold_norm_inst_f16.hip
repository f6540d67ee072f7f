// fold_norm_inst_f16.hip -- instantiates the norms around a block for f16 rows and parameters.
#include "fold_norm_kernel.h"

namespace pccl_dev {
PCCL_DEFINE_FOLD_NORM(PCCL_F16, false)
}  // namespace pccl_dev
