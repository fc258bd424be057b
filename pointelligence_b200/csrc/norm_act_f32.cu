// The group norm with activation and dropout for rows of f32.
#include "norm_act.cuh"

namespace pcx {
template int norm_act_rows<float>(const NormAct &, int, bool, cudaStream_t);
}
