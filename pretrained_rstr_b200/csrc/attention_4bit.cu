// Causal attention over a cache held in 4 bits: the launch, and the bfloat16 form of the kernel in attention_4bit.cuh.
#include "attention_4bit.cuh"

int prb_attention_4bit_f32(attn4::Args p, cudaStream_t stream);   // attention_4bit_f32.cu

namespace {
using namespace attn4;

template <bool LOW> int launch_by(const Args& p, cudaStream_t stream) {
    switch (cache4::groups_of(p.head_dim)) {
        case 1: return launch_one<1, LOW, __nv_bfloat16>(p, stream);
        case 2: return launch_one<2, LOW, __nv_bfloat16>(p, stream);
        case 3: return launch_one<3, LOW, __nv_bfloat16>(p, stream);
        default: return launch_one<4, LOW, __nv_bfloat16>(p, stream);
    }
}

// Parts of a unit's keys: as many as give every SM about four CTAs (of four warps each), each with a stage a warp at
// least.
int parts_for(long units, int max_context, int window, int ng) {
    const int sk = stage_keys(ng);
    const int span = window > 0 && window < max_context ? window + sk : max_context;
    const int stages = (span + sk - 1) / sk;
    int parts = 1;
    while (parts < MAX_PARTS && units * parts * 2 <= 4L * prb_sm_count() && stages >= parts * 2 * WARPS) parts *= 2;
    return parts;
}
}  // namespace

// tile_most: the most tokens a tile has.  max_context: the most positions a request holds after the step.
PRB_API int prb_attention_4bit(void* out, long out_stride, const void* q, long q_stride, const void* k_tiles,
                               const void* v_tiles, const int* block_table, const int* positions, const int* tile_req,
                               const int* tile_row0, const int* tile_rows, const int* tile_count, int n_tiles,
                               int tile_most, int n_tokens, int n_requests, int heads, int kv_heads, int head_dim,
                               int page_size, int max_pages, int num_pages, float scale, int window, int max_context,
                               int parts, int dtype, int* status, cudaStream_t stream) {
    if (n_tiles <= 0 || n_tokens <= 0) return 0;
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || tile_most <= 0 || !cache4::takes(head_dim, page_size) ||
        max_pages <= 0 || num_pages <= 0 || n_requests <= 0 || (long)max_pages * page_size > 0x7fffffffL)
        return PRB_E_SIZE;
    if (window < 0 || max_context <= 0 || parts < 0 || parts > MAX_PARTS) return PRB_E_ARG;
    if ((uintptr_t)k_tiles % 16 != 0 || (uintptr_t)v_tiles % 16 != 0) return PRB_E_ALIGN;
    if (dtype != PRB_F32 && dtype != PRB_BF16) return PRB_E_DTYPE;
    const int size = dtype == PRB_F32 ? 4 : 2, ng = cache4::groups_of(head_dim), hpg = heads / kv_heads;
    Args p{};
    p.out = out; p.out_stride = out_stride; p.q = q; p.q_stride = q_stride;
    p.k_tiles = (const uint8_t*)k_tiles; p.v_tiles = (const uint8_t*)v_tiles;
    p.block_table = block_table; p.positions = positions;
    p.tile_req = tile_req; p.tile_row0 = tile_row0; p.tile_rows = tile_rows; p.tile_count = tile_count;
    p.n_tokens = n_tokens; p.n_requests = n_requests; p.n_tiles = n_tiles;
    p.heads = heads; p.kv_heads = kv_heads; p.hpg = hpg;
    p.head_dim = head_dim; p.page_size = page_size;
    p.piece = page_size;
    const int sk = stage_keys(ng);
    if (page_size > sk || sk % page_size != 0) p.piece = page_size % sk == 0 ? sk : page_size % 32 == 0 ? 32 : 16;
    p.max_pages = max_pages; p.num_pages = num_pages;
    p.tile_bytes = cache4::tile_bytes(head_dim, page_size);
    p.scale = scale; p.window = window;
    p.wide = (uintptr_t)q % 16 == 0 && (q_stride * size) % 16 == 0;
    p.status = status;
    const long rows = (long)tile_most * hpg;
    const bool low = dtype == PRB_F32 || rows <= 8;
    const long subs = (rows + (low ? 7 : 15)) / (low ? 8 : 16);
    const long units = (long)n_tiles * kv_heads * subs;
    if (units > 0x7fffffffL / MAX_PARTS) return PRB_E_SIZE;
    p.subs = (int)subs;
    p.parts = parts > 0 ? parts : parts_for(units, max_context, window, ng);
    if (dtype == PRB_F32) return prb_attention_4bit_f32(p, stream);
    return low ? launch_by<true>(p, stream) : launch_by<false>(p, stream);
}
