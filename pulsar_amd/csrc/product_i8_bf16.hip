// product_i8_bf16.hip - the kernels of pulsar_matmul_i8 whose rows are bf16.
#include "pk_i8_launch.h"

template int pk::launch_i8<PULSAR_TYPE_BF16>(const pk::I8Args &);
