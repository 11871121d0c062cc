// The float32 form of the attention over a cache held in 4 bits (the kernel is in attention_4bit.cuh).
#include "attention_4bit.cuh"

int prb_attention_4bit_f32(const attn4::Args& p, long rows, int max_context, int parts, cudaStream_t stream) {
    switch (cache4::groups_of(p.head_dim)) {
        case 1:
            return rows <= 8 ? attn4::launch_by<1, 1, float>(p, rows, max_context, parts, stream)
                             : attn4::launch_by<1, 2, float>(p, rows, max_context, parts, stream);
        case 2:
            return rows <= 8 ? attn4::launch_by<2, 1, float>(p, rows, max_context, parts, stream)
                             : attn4::launch_by<2, 2, float>(p, rows, max_context, parts, stream);
        case 3:
            return rows <= 8 ? attn4::launch_by<3, 1, float>(p, rows, max_context, parts, stream)
                             : attn4::launch_by<3, 2, float>(p, rows, max_context, parts, stream);
        default: return attn4::launch_by<4, 1, float>(p, rows, max_context, parts, stream);
    }
}
