// The products by expert of f16 rows.
#include "prod_launch.h"

namespace ktmi {

ProdTable prod_table_f16() {
  return {&ProdOps<F16>::tile,      &ProdOps<F16>::sum,     &ProdOps<F16>::rows,
          &launch_fp8_tile<F16>, &launch_quantise<F16>, &launch_gated_grad<F16>};
}

}  // namespace ktmi
