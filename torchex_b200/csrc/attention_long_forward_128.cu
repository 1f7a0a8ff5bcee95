#include "attention_long_forward.cuh"

namespace texb {
namespace attention {
template int long_forward_by_type<128>(const Problem&, int, int, cudaStream_t);
template int long_forward_timeouts<128>(int*);
}  // namespace attention
}  // namespace texb
