// The float32 form of the attention over a cache held in 4 bits (the kernel is in attention_4bit.cuh).
#include "attention_4bit.cuh"

namespace {
template <int NG> int by(const attn4::Args& p, long rows, int max_context, int parts, cudaStream_t stream) {
    if (rows <= 4) return attn4::launch_by<NG, 1, 1, float>(p, rows, max_context, parts, stream);
    // (16 rows' queries in three pieces fit the registers up to two groups)
    if (rows <= 8 || NG > 2) return attn4::launch_by<NG, 1, 2, float>(p, rows, max_context, parts, stream);
    return attn4::launch_by<NG, (NG > 2 ? 1 : 2), 2, float>(p, rows, max_context, parts, stream);
}
}  // namespace

int prb_attention_4bit_f32(const attn4::Args& p, long rows, int max_context, int parts, cudaStream_t stream) {
    switch (cache4::groups_of(p.head_dim)) {
        case 1: return by<1>(p, rows, max_context, parts, stream);
        case 2: return by<2>(p, rows, max_context, parts, stream);
        case 3: return by<3>(p, rows, max_context, parts, stream);
        default: return by<4>(p, rows, max_context, parts, stream);
    }
}
