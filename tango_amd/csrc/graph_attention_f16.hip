// The attention kernels of graph_attention.hpp for fp16 results (one file a type: they compile side by side).
#include "graph_attention.hpp"

namespace tango {

template bool launch_attention<f16_t, f16_t>(AttnPass, AttnArgs, JoinArgs, int64_t, bool, hipStream_t);
template bool launch_attention<int8_t, f16_t>(AttnPass, AttnArgs, JoinArgs, int64_t, bool, hipStream_t);

}  // namespace tango
