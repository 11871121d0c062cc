// Causal attention over a cache held in 4 bits: the launch, and the bfloat16 form of the kernel in attention_4bit.cuh.
#include "attention_4bit.cuh"
#include "ranges.cuh"

// (attention_4bit_tile.cu, attention_4bit_f32.cu, attention_4bit_rows.cu)
bool prb_attention_4bit_tile_takes(int head_dim, int page_size, int window, const void* q, long q_stride, const void* out,
                                   long out_stride);
int prb_attention_4bit_tile(void* out, long out_stride, const void* q, long q_stride, const uint8_t* k_tiles,
                            const uint8_t* v_tiles, const int* block_table, const int* positions, const int* tile_req,
                            const int* tile_row0, const int* tile_rows, const int* tile_count, int n_tiles, long rows,
                            int n_tokens, int n_requests, int kv_heads, int hpg, int head_dim, int page_size, int max_pages,
                            int num_pages, float scale, int max_context, int parts, int* status, cudaStream_t stream);
int prb_attention_4bit_f32(const attn4::Args& p, long rows, int max_context, int parts, cudaStream_t stream);
int prb_attention_4bit_rows(const attn4::Args& p, long rows, int max_context, int parts, cudaStream_t stream);

namespace {
// More rows than this go to the tensor-memory kernel where it takes the call: 33 tokens at 300 of 12 heads of 64 20.8 us by
// the other one, 12.6 by that; 8 x 33 at 1,000 33.7 and 25.3; 16 x 64 at 500 of 16 heads 49.8 and 25.1; 20 x 12 tokens at
// 1,000 of 4 heads a key/value head of 128 61.4 and 46.4.
constexpr long TILE_ROWS = 32;

// up to 4 rows a tile, or 8
template <int NG> int by(const attn4::Args& p, long rows, int max_context, int parts, cudaStream_t stream) {
    return rows <= 4 ? attn4::launch_by<NG, 1, 1, __nv_bfloat16>(p, rows, max_context, parts, stream)
                     : attn4::launch_by<NG, 1, 2, __nv_bfloat16>(p, rows, max_context, parts, stream);
}
int launch_few(const attn4::Args& p, long rows, int max_context, int parts, cudaStream_t stream) {
    switch (cache4::groups_of(p.head_dim)) {
        case 1: return by<1>(p, rows, max_context, parts, stream);
        case 2: return by<2>(p, rows, max_context, parts, stream);
        case 3: return by<3>(p, rows, max_context, parts, stream);
        default: return by<4>(p, rows, max_context, parts, stream);
    }
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
    if (window < 0 || max_context <= 0 || parts < 0 || parts > attn4::MAX_PARTS ||
        !(scale > 0.0f && scale <= 1e37f))                   // (scores are masked and compared before they are scaled)
        return PRB_E_ARG;
    if ((uintptr_t)k_tiles % 16 != 0 || (uintptr_t)v_tiles % 16 != 0) return PRB_E_ALIGN;
    if (dtype != PRB_F32 && dtype != PRB_BF16) return PRB_E_DTYPE;
    const int size = dtype == PRB_F32 ? 4 : 2, hpg = heads / kv_heads;
    const long width = (long)heads * head_dim * size, word = sizeof(int);
    const long pool = num_pages * (long)kv_heads * cache4::tile_bytes(head_dim, page_size);
    const PrbRange rows_out{out, prb_span(n_tokens, out_stride * size, width)}, said{status, 4 * word};
    const PrbRange queries{q, prb_span(n_tokens, q_stride * size, width)}, keys{k_tiles, pool}, values{v_tiles, pool};
    const PrbRange table{block_table, (long)n_requests * max_pages * word}, places{positions, n_tokens * word};
    const PrbRange reqs{tile_req, n_tiles * word}, firsts{tile_row0, n_tiles * word}, counts{tile_rows, n_tiles * word};
    if (!prb_rows_apart(out, out_stride * size, q, q_stride * size, n_tokens, width) ||
        !prb_apart({rows_out, said}, {keys, values, table, places, reqs, firsts, counts, {tile_count, word}}) ||
        prb_overlap(said, queries))
        return PRB_E_OVERLAP;
    attn4::Args p{};
    p.out = out; p.out_stride = out_stride; p.q = q; p.q_stride = q_stride;
    p.k_tiles = (const uint8_t*)k_tiles; p.v_tiles = (const uint8_t*)v_tiles;
    p.block_table = block_table; p.positions = positions;
    p.tile_req = tile_req; p.tile_row0 = tile_row0; p.tile_rows = tile_rows; p.tile_count = tile_count;
    p.n_tokens = n_tokens; p.n_requests = n_requests; p.n_tiles = n_tiles; p.tile_most = tile_most;
    p.heads = heads; p.kv_heads = kv_heads; p.hpg = hpg;
    p.head_dim = head_dim; p.page_size = page_size;
    p.max_pages = max_pages; p.num_pages = num_pages;
    p.tile_bytes = cache4::tile_bytes(head_dim, page_size);
    p.scale = scale; p.window = window;
    p.wide = (uintptr_t)q % 16 == 0 && (q_stride * size) % 16 == 0;
    p.status = status;
    p.magic = 0x43004300u;
    const long rows = (long)tile_most * hpg;
    if (dtype == PRB_F32) return prb_attention_4bit_f32(p, rows, max_context, parts, stream);
    if (rows > TILE_ROWS && prb_attention_4bit_tile_takes(head_dim, page_size, window, q, q_stride, out, out_stride))
        return prb_attention_4bit_tile(out, out_stride, q, q_stride, p.k_tiles, p.v_tiles, block_table, positions, tile_req,
                                       tile_row0, tile_rows, tile_count, n_tiles, rows, n_tokens, n_requests, kv_heads, hpg,
                                       head_dim, page_size, max_pages, num_pages, scale, max_context, parts, status, stream);
    return rows <= 8 ? launch_few(p, rows, max_context, parts, stream)
                     : prb_attention_4bit_rows(p, rows, max_context, parts, stream);
}
