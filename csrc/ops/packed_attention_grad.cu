#include "packed.hpp"
namespace mccl { namespace ops { cudaError_t packed_attention_grad(const PackedAttentionGradArgs&, cudaStream_t) { return cudaErrorNotSupported; } } }
