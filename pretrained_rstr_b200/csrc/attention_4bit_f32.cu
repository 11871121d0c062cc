// The float32 form of the attention over a cache held in 4 bits (the kernel is in attention_4bit.cuh).
#include "attention_4bit.cuh"

int prb_attention_4bit_f32(attn4::Args p, cudaStream_t stream) {
    using namespace attn4;
    switch (cache4::groups_of(p.head_dim)) {
        case 1: return launch_one<1, true, float>(p, stream);
        case 2: return launch_one<2, true, float>(p, stream);
        case 3: return launch_one<3, true, float>(p, stream);
        default: return launch_one<4, true, float>(p, stream);
    }
}
