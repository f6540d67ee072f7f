// fold_norm_inst_bf16.hip -- instantiates the norms around a block for bf16 rows and parameters.
#include "fold_norm_kernel.h"

namespace pccl_dev {
PCCL_DEFINE_FOLD_NORM(PCCL_BF16, false)
}  // namespace pccl_dev
