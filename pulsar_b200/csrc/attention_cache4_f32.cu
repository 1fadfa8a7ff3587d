// The float32 kernels of attention over a cache of 4 bits (attention_cache4.cuh).
#include "attention_cache4.cuh"

namespace pb {

int attend_4bit_f32(const Attend4& a, int groups, int rows, int most_tokens, cudaStream_t stream) {
    return launch_attend_4bit_of<float>(a, groups, rows, most_tokens, stream);
}

}  // namespace pb
