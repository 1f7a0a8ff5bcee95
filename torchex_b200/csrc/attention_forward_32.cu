#include "attention_forward.cuh"

namespace texb {
namespace attention {
template int forward_by_type<32>(const Problem&, int, int, cudaStream_t);
}  // namespace attention
}  // namespace texb
