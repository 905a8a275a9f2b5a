// The products by expert of bf16 rows.
#include "prod_launch.h"

namespace ktmi {

ProdTable prod_table_bf16() {
  return {&ProdOps<BF16>::tile,      &ProdOps<BF16>::sum,     &ProdOps<BF16>::rows,
          &launch_fp8_tile<BF16>, &launch_quantise<BF16>, &launch_gated_grad<BF16>};
}

}  // namespace ktmi
