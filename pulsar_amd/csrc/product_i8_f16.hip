// product_i8_f16.hip - the kernels of pulsar_matmul_i8 whose rows are f16.
#include "pk_i8_launch.h"

template int pk::launch_i8<PULSAR_TYPE_F16>(const pk::I8Args &);
