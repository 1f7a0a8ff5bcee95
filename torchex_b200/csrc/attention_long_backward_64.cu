#include "attention_long_backward.cuh"

namespace texb {
namespace attention {
template int long_backward_by_type<64>(const Problem&, int, int, cudaStream_t);
template int long_backward_timeouts<64>(int*);
}  // namespace attention
}  // namespace texb
