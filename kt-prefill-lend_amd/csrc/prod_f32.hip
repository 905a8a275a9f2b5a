// The products by expert of f32 rows.
#include "prod_launch.h"

namespace ktmi {

ProdTable prod_table_f32() {
  return {&ProdOps<F32>::tile,      &ProdOps<F32>::sum,     &ProdOps<F32>::rows,
          &launch_fp8_tile<F32>, &launch_quantise<F32>, &launch_gated_grad<F32>};
}

}  // namespace ktmi
