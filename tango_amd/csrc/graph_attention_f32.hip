// The attention kernels of graph_attention.hpp for fp32 results (one file a type: they compile side by side).
#include "graph_attention.hpp"

namespace tango {

template bool launch_attention<float, float>(AttnPass, AttnArgs, JoinArgs, int64_t, bool, hipStream_t);
template bool launch_attention<int8_t, float>(AttnPass, AttnArgs, JoinArgs, int64_t, bool, hipStream_t);

}  // namespace tango
