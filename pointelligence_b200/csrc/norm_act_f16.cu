// The group norm with activation and dropout for rows of f16.
#include "norm_act.cuh"

namespace pcx {
template int norm_act_rows<__half>(const NormAct &, int, bool, cudaStream_t);
}
