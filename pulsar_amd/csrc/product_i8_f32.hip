// product_i8_f32.hip - the kernels of pulsar_matmul_i8 whose rows are f32.
#include "pk_i8_launch.h"

template int pk::launch_i8<PULSAR_TYPE_F32>(const pk::I8Args &);
