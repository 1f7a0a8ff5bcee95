#include "attention_backward.cuh"

namespace texb {
namespace attention {
template int backward_by_type<128>(const Problem&, int, int, cudaStream_t);
}  // namespace attention
}  // namespace texb
