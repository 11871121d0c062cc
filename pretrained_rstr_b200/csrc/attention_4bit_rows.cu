// The attention over a cache held in 4 bits for tiles of more than 8 rows (the kernel is in attention_4bit.cuh): 16 rows a
// CTA, or 32, where the turning of codes into operands is shared by four products' columns (with more than two groups
// 32 rows' results would not fit the registers).
#include "attention_4bit.cuh"

int prb_attention_4bit_rows(const attn4::Args& p, long rows, int max_context, int parts, cudaStream_t stream) {
    switch (cache4::groups_of(p.head_dim)) {
        case 1:
            return rows <= 16 ? attn4::launch_by<1, 2, 2, __nv_bfloat16>(p, rows, max_context, parts, stream)
                              : attn4::launch_by<1, 4, 2, __nv_bfloat16>(p, rows, max_context, parts, stream);
        case 2:
            return rows <= 16 ? attn4::launch_by<2, 2, 2, __nv_bfloat16>(p, rows, max_context, parts, stream)
                              : attn4::launch_by<2, 4, 2, __nv_bfloat16>(p, rows, max_context, parts, stream);
        case 3:
            return attn4::launch_by<3, 2, 2, __nv_bfloat16>(p, rows, max_context, parts, stream);
        default:
            return attn4::launch_by<4, 2, 2, __nv_bfloat16>(p, rows, max_context, parts, stream);
    }
}
