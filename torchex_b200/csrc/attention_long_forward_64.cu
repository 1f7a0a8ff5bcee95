#include "attention_long_forward.cuh"

namespace texb {
namespace attention {
template int long_forward_by_type<64>(const Problem&, int, int, cudaStream_t);
template int long_forward_timeouts<64>(int*);
}  // namespace attention
}  // namespace texb
