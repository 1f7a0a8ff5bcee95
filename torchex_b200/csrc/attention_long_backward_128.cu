#include "attention_long_backward.cuh"

namespace texb {
namespace attention {
template int long_backward_by_type<128>(const Problem&, int, int, cudaStream_t);
template int long_backward_timeouts<128>(int*);
}  // namespace attention
}  // namespace texb
