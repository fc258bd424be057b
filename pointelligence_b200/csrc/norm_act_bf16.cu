// The group norm with activation and dropout for rows of bf16.
#include "norm_act.cuh"

namespace pcx {
template int norm_act_rows<__nv_bfloat16>(const NormAct &, int, bool, cudaStream_t);
}
