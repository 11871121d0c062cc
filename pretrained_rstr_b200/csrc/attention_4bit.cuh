// Causal attention over a cache held in 4 bits (cache4.cuh): the kernel that takes every tile of tokens, single
// ones and a few drafted ones above all.  Instantiated in attention_4bit.cu (bfloat16) and attention_4bit_f32.cu.
//
// With k = middle + step * (c - 8) per group g of 32 channels, a score is
//     q . k = sum over g of  step_g * (q_g . (c_g - 8)) + middle_g * (sum of q_g)
// and a result is
//     sum over keys of  (p * step_g) * (c - 8)  +  sum over keys of p * middle_g.
// The codes less 8 are whole numbers from -8 to 7, exact in bfloat16, so the cache is never turned into rounded
// numbers: the products run on the matrix units (mma.sync, 16 x 8 x 16) with the codes as one operand, and the
// steps and middles join in 32 bits.  bfloat16 queries are exact too, and p * step is the one rounding (2^-8,
// as probabilities are rounded before any such product).  float32 queries, and then p * step, go as the sum of
// three bfloat16 numbers (24 bits), which makes three products of 32-bit exactness.
//
// What bounds it: the bytes of the cache where there is one row a key/value head, the instructions that turn words of
// codes into operands beside them (11 a word of 8 codes), the products from some rows on.
//
// One CTA of four warps takes up to 16 rows (8 in the LOW form; a row is a token and one of the heads that share keys
// and values) of one tile for one key/value head, or one of S parts of their keys; the parts are a cluster, whose
// CTAs meet through distributed shared memory, so there is no workspace and no counter, and parts are added in the
// keys' order whatever came first.  Each warp takes every fourth stage of SK keys and keeps two stages of its own in
// flight (bulk copies, no multicast, of whole tiles where a page is a stage).  Nothing is shared between warps until
// the end.
#pragma once
#include "cache4.cuh"
#include "tcgen05.cuh"

namespace attn4 {
using namespace tc5;

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int STAGES = 2;                  // ring buffers of a warp
constexpr int MAX_PARTS = 8;               // CTAs of a cluster (portable)

// keys of a stage: 64, or 32 where four groups would make a warp's two buffers larger than an SM likes
__host__ __device__ constexpr int stage_keys(int ng) { return ng <= 2 ? 64 : 32; }

struct Args {
    void* out;
    long out_stride;
    const void* q;
    long q_stride;
    const uint8_t* k_tiles;
    const uint8_t* v_tiles;
    const int* block_table;
    const int* positions;
    const int* tile_req;
    const int* tile_row0;
    const int* tile_rows;
    const int* tile_count;                 // null: every tile of the launch
    int n_tokens;                          // rows of q and out
    int n_requests;                        // rows of the block table
    int n_tiles, subs, parts;
    int heads, kv_heads, hpg;              // hpg: query heads per key/value head
    int head_dim, page_size, piece;        // piece: keys that lie together in a page and in a stage
    int max_pages, num_pages;
    int tile_bytes;
    float scale;
    int window;
    int wide;                              // queries can be read 16 bytes at a time
    int* status;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes i and i + 4 of a word, less 8, as two bfloat16 numbers: 0x4300 | c is 128 + c.
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int i) {
    const uint32_t u = ((word >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 off = __floats2bfloat162_rn(136.0f, 136.0f);
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), off);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lds_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// x as the sum of PIECES bfloat16 numbers, two x at a time.
template <int PIECES> __device__ __forceinline__ void split2(float x, float y, uint32_t (&out)[PIECES]) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        out[i] = *reinterpret_cast<const uint32_t*>(&h);
        if (i + 1 < PIECES) {
            x -= __low2float(h);
            y -= __high2float(h);
        }
    }
}

template <int NG> struct Layout {
    static constexpr int SK = stage_keys(NG);
    static constexpr int KIND = SK * (16 * NG + 4 * NG);      // most bytes of a stage's keys (and of its values)
    static constexpr int STAGE = 2 * KIND;
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int BARS = WARPS * STAGES * 8;
};

template <int NG, bool LOW, typename T>
__global__ void __launch_bounds__(THREADS) attention_4bit_kernel(const Args p) {
    using L = Layout<NG>;
    constexpr int SK = L::SK, ROWS = LOW ? 8 : 16, NT = SK / 8, RH = LOW ? 1 : 2;
    constexpr int PIECES = sizeof(T) == 4 ? 3 : 1;
    constexpr int DP = NG * 32, PART = DP + 2;                // floats a row of a partial state: values, maximum, sum
    extern __shared__ __align__(128) uint8_t smem[];
    static_assert(ROWS * PART * 4 <= STAGES * L::STAGE, "a warp's state fits its own ring");
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::RING);
    volatile int* failed = reinterpret_cast<volatile int*>(smem + L::RING + L::BARS);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = lane >> 2, j = lane & 3;
    prb_grid_launch_dependents();
    if (threadIdx.x < WARPS * STAGES) mbar_init(smem_u32(&bars[threadIdx.x]), 1);
    if (threadIdx.x == 0) *failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    prb_grid_wait();

    // ---------------------------------------------------------------- which rows, which keys
    const int unit = blockIdx.x / p.parts, rank = blockIdx.x - unit * p.parts;
    const int per = p.kv_heads * p.subs;
    const int tile = unit / per;
    const int hk = (unit - tile * per) / p.subs, sub = unit - tile * per - hk * p.subs;
    const int n_tiles = p.tile_count != nullptr ? min(*p.tile_count, p.n_tiles) : p.n_tiles;
    // (the same answer for all CTAs of a cluster, whose unit is one)
    if (tile >= n_tiles) return;
    const int req = p.tile_req[tile], row0 = p.tile_row0[tile], tokens = p.tile_rows[tile];
    const int first = sub * ROWS;                             // first row of this unit among the tile's
    if (tokens <= 0 || first >= tokens * p.hpg) return;
    const bool placed = req >= 0 && req < p.n_requests && row0 >= 0 && tokens <= p.n_tokens && row0 <= p.n_tokens - tokens;
    const int pos0 = placed ? p.positions[row0] : -1;
    if (pos0 < 0 || pos0 > p.max_pages * p.page_size - tokens || tokens * p.hpg > p.subs * ROWS) {
        if (threadIdx.x == 0 && rank == 0) prb_set_status(p.status, PRB_S_POSITION_RANGE, row0, pos0, tokens);
        return;
    }
    const int rows = min(ROWS, tokens * p.hpg - first);
    const int pos_lo = pos0 + first / p.hpg, pos_hi = pos0 + (first + rows - 1) / p.hpg;
    const int key_lo = p.window > 0 ? max(0, pos_lo - p.window + 1) : 0;
    const int blk_lo = key_lo / SK, n_blk = pos_hi / SK - blk_lo + 1;
    const int my_lo = blk_lo + (int)((long)n_blk * rank / p.parts);
    const int my_hi = blk_lo + (int)((long)n_blk * (rank + 1) / p.parts);
    const int* table = p.block_table + (size_t)req * p.max_pages;

    // ---------------------------------------------------------------------- queries
    // Channel order of the reduction: thread j of a quad has channels 8 j + (i, i + 4), the codes that one shift and
    // one mask take from word j.
    uint32_t qa[NG][2][PIECES][2 * RH];                       // [group][half of the reduction][piece][operand]
    float qsum[NG][RH];
#pragma unroll
    for (int r = 0; r < RH; ++r) {
        const int row = n + 8 * r, at = first + min(row, rows - 1);
        const int tk = at / p.hpg, h = hk * p.hpg + at - tk * p.hpg;
        const T* src = reinterpret_cast<const T*>(p.q) + (long)(row0 + tk) * p.q_stride + (long)h * p.head_dim;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int c0 = g * 32 + j * 8;
            float x[8];
            if (row < rows && c0 < p.head_dim) {
                if (p.wide) {
                    if (sizeof(T) == 2) {
                        const uint4 w = *reinterpret_cast<const uint4*>(src + c0);
                        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[2 * i] = __uint_as_float(ww[i] << 16);
                            x[2 * i + 1] = __uint_as_float(ww[i] & 0xffff0000u);
                        }
                    } else {
                        const float4 a = *reinterpret_cast<const float4*>(src + c0);
                        const float4 b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src + c0) + 4);
                        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
                        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = prb_to_float<T>(src[c0 + i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = 0.0f;
            }
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += x[i];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            qsum[g][r] = sum;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w[PIECES];
                split2<PIECES>(x[i], x[i + 4], w);
#pragma unroll
                for (int z = 0; z < PIECES; ++z) qa[g][i >> 1][z][(i & 1) * RH + r] = w[z];
            }
        }
    }

    // ------------------------------------------------------------------------ stages
    const uint32_t ring = smem_u32(smem) + warp * STAGES * L::STAGE;
    const uint8_t* ring_p = smem + warp * STAGES * L::STAGE;
    const uint32_t bar0 = smem_u32(&bars[warp * STAGES]);
    const int pieces = SK / p.piece;
    const int piece_bytes = p.piece * (p.head_dim / 2 + 4 * NG);
    const int codes_of_page = p.page_size * (p.head_dim / 2);
    const bool whole = p.piece == p.page_size;
    // Lane i looks after piece i of a stage: its page, ahead of time, and its copies.
    auto page_of = [&](int blk) -> int {
        const int key = blk * SK + lane * p.piece;
        if (blk >= my_hi || lane >= pieces || key > pos_hi || key + p.piece <= key_lo) return -2;    // nothing to fetch
        return table[key / p.page_size];
    };
    auto request = [&](int blk, int st, int page) {
        bool fetch = page != -2;
        if (fetch && (page < 0 || page >= p.num_pages)) {
            // (recorded; the stage keeps what it held, and the tile's result is not to be used)
            prb_set_status(p.status, PRB_S_PAGE_RANGE, row0, blk * SK + lane * p.piece, page);
            fetch = false;
        }
        const unsigned who = __ballot_sync(0xffffffffu, fetch);
        const uint32_t bar = bar0 + st * 8;
        if (lane == 0) mbar_expect_tx(bar, (uint32_t)(__popc(who) * 2 * piece_bytes));
        __syncwarp();
        if (!fetch) return;
        const int at = (blk * SK + lane * p.piece) % p.page_size;
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            const uint8_t* src = (kind ? p.v_tiles : p.k_tiles) + ((size_t)page * p.kv_heads + hk) * (size_t)p.tile_bytes;
            uint32_t dst = ring + st * L::STAGE + kind * L::KIND + lane * piece_bytes;
            if (whole) {
                bulk_load(dst, src, piece_bytes, bar);
            } else {
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const int row = min(16, (p.head_dim - g * 32) / 2);
                    bulk_load(dst, src + g * p.page_size * 16 + at * row, p.piece * row, bar);
                    dst += p.piece * row;
                }
                bulk_load(dst, src + codes_of_page + at * NG * 4, p.piece * NG * 4, bar);
            }
        }
    };

    float o[NG][4][4];
    float mid[NG][RH], m[RH], l[RH];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[g][i][e] = 0.0f;
#pragma unroll
        for (int r = 0; r < RH; ++r) mid[g][r] = 0.0f;
    }
#pragma unroll
    for (int r = 0; r < RH; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
    }
    const float sl2 = p.scale * 1.4426950408889634f;          // scores are handled in log2 units
    // (the short last group's rows are 8 bytes apart; its words 2 and 3 do not exist: words 0 and 1 stand in, against
    // queries of zero and for channels that are not stored)
    const bool short_last = p.head_dim % 32 != 0;

#pragma unroll
    for (int st = 0; st < STAGES; ++st) {
        const int blk = my_lo + warp + st * WARPS;
        if (blk < my_hi) request(blk, st, page_of(blk));
    }
    int ahead = page_of(my_lo + warp + STAGES * WARPS);
    bool alive = true;
    int it = 0;
    for (int blk = my_lo + warp; blk < my_hi; blk += WARPS, ++it) {
        const int st = it % STAGES;
        alive = mbar_wait_warp(bar0 + st * 8, (it / STAGES) & 1, failed);
        if (!alive) {
            if (lane == 0) prb_set_status(p.status, PRB_S_WAIT_TIMEOUT, 41, blockIdx.x, blk);
            break;
        }
        const uint8_t* ks = ring_p + st * L::STAGE;
        const uint8_t* vs = ks + L::KIND;
        const int key0 = blk * SK;
        const bool masked = key0 + SK - 1 > pos_lo || (p.window > 0 && key0 <= pos_hi - p.window);
        // ---- scores
        float s[NT][2 * RH];
#pragma unroll
        for (int c = 0; c < SK / 16; ++c) {
            const int pc = (c * 16) / p.piece, in = c * 16 - pc * p.piece;
            const uint8_t* base = ks + pc * piece_bytes;
            const uint8_t* par = base + p.piece * (p.head_dim / 2) + in * NG * 4;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float (&sc)[2 * RH] = s[2 * c + t];
#pragma unroll
                for (int e = 0; e < 2 * RH; ++e) sc[e] = 0.0f;
                uint32_t pr[2][NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    pr[0][g] = *reinterpret_cast<const uint32_t*>(par + ((t * 8 + 2 * j) * NG + g) * 4);
                    pr[1][g] = *reinterpret_cast<const uint32_t*>(par + ((t * 8 + 2 * j + 1) * NG + g) * 4);
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const bool sh = g == NG - 1 && short_last;
                    const int off = sh ? (in + t * 8 + n) * 8 + (j & 1) * 4 : (in + t * 8 + n) * 16 + j * 4;
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(base + g * p.piece * 16 + off);
                    const uint32_t b0 = code_pair(w, 0), b1 = code_pair(w, 1), b2 = code_pair(w, 2), b3 = code_pair(w, 3);
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int z = PIECES - 1; z >= 0; --z) {
                        if (LOW) {
                            mma(acc, qa[g][0][z][0], 0u, qa[g][0][z][RH], 0u, b0, b1);
                            mma(acc, qa[g][1][z][0], 0u, qa[g][1][z][RH], 0u, b2, b3);
                        } else {
                            mma(acc, qa[g][0][z][0], qa[g][0][z][1 % (2 * RH)], qa[g][0][z][RH], qa[g][0][z][(RH + 1) % (2 * RH)], b0, b1);
                            mma(acc, qa[g][1][z][0], qa[g][1][z][1 % (2 * RH)], qa[g][1][z][RH], qa[g][1][z][(RH + 1) % (2 * RH)], b2, b3);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < RH; ++r)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float step = __uint_as_float(pr[e][g] << 16);
                            const float middle = __uint_as_float(pr[e][g] & 0xffff0000u);
                            sc[2 * r + e] = fmaf(step, acc[2 * r + e], fmaf(middle, qsum[g][r], sc[2 * r + e]));
                        }
                }
            }
        }
        // ---- mask, maximum, exponentials
        float alpha[RH];
#pragma unroll
        for (int r = 0; r < RH; ++r) {
            const int row = n + 8 * r;
            const int pos = pos0 + (first + min(row, rows - 1)) / p.hpg;
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float v = s[t][2 * r + e] * sl2;
                    if (masked) {
                        const int key = key0 + t * 8 + 2 * j + e;
                        if (key > pos || (p.window > 0 && key <= pos - p.window)) v = -INFINITY;
                    }
                    s[t][2 * r + e] = v;
                    top = fmaxf(top, v);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float now = fmaxf(m[r], top);
            const float ref = now == -INFINITY ? 0.0f : now;
            alpha[r] = exp2_fast(m[r] - ref);                 // (0 while nothing was seen)
            m[r] = now;
            float sum = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[t][2 * r + e] = exp2_fast(s[t][2 * r + e] - ref);
                    sum += s[t][2 * r + e];
                }
            l[r] = l[r] * alpha[r] + sum;
        }
        bool moved = alpha[0] != 1.0f;
        if (RH == 2) moved = moved || alpha[RH - 1] != 1.0f;
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
#pragma unroll
                for (int r = 0; r < RH; ++r) mid[g][r] *= alpha[r];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < RH; ++r) {
                        o[g][i][2 * r] *= alpha[r];
                        o[g][i][2 * r + 1] *= alpha[r];
                    }
            }
        }
        // ---- values
#pragma unroll
        for (int c = 0; c < SK / 16; ++c) {
            const int pc = (c * 16) / p.piece, in = c * 16 - pc * p.piece;
            const uint8_t* base = vs + pc * piece_bytes;
            const uint8_t* par = base + p.piece * (p.head_dim / 2) + in * NG * 4;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                // p * step of keys 2 j, 2 j + 1 (tile 0) and 8 + 2 j, 9 + 2 j (tile 1)
                uint32_t a[PIECES][2][RH];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t p0 = *reinterpret_cast<const uint32_t*>(par + ((t * 8 + 2 * j) * NG + g) * 4);
                    const uint32_t p1 = *reinterpret_cast<const uint32_t*>(par + ((t * 8 + 2 * j + 1) * NG + g) * 4);
#pragma unroll
                    for (int r = 0; r < RH; ++r) {
                        const float w0 = s[2 * c + t][2 * r], w1 = s[2 * c + t][2 * r + 1];
                        float x0 = w0 * __uint_as_float(p0 << 16), x1 = w1 * __uint_as_float(p1 << 16);
                        float y0 = w0 * __uint_as_float(p0 & 0xffff0000u), y1 = w1 * __uint_as_float(p1 & 0xffff0000u);
                        if (masked) {
                            // (a masked key's step and middle may be anything, NaN too)
                            if (w0 == 0.0f) x0 = y0 = 0.0f;
                            if (w1 == 0.0f) x1 = y1 = 0.0f;
                        }
                        mid[g][r] += y0 + y1;
                        uint32_t w[PIECES];
                        split2<PIECES>(x0, x1, w);
#pragma unroll
                        for (int z = 0; z < PIECES; ++z) a[z][t][r] = w[z];
                    }
                }
                const bool sh = g == NG - 1 && short_last;
                const uint8_t* col = base + g * p.piece * 16 + (sh ? (n & 1) * 4 : (n & 3) * 4) + (n >> 2) * 2;
                const int row = sh ? 8 : 16;
                auto half = [&](int key) -> uint32_t { return *reinterpret_cast<const uint16_t*>(col + (in + key) * row); };
                const uint32_t u = half(2 * j) | (half(2 * j + 1) << 16);
                const uint32_t v = half(8 + 2 * j) | (half(9 + 2 * j) << 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t b0 = code_pair(u, i), b1 = code_pair(v, i);
#pragma unroll
                    for (int z = PIECES - 1; z >= 0; --z) {
                        if (LOW)
                            mma(o[g][i], a[z][0][0], 0u, a[z][1][0], 0u, b0, b1);
                        else
                            mma(o[g][i], a[z][0][0], a[z][0][RH - 1], a[z][1][0], a[z][1][RH - 1], b0, b1);
                    }
                }
            }
        }
        __syncwarp();                                          // every lane has read the stage
        if (blk + STAGES * WARPS < my_hi) {
            request(blk + STAGES * WARPS, st, ahead);
            ahead = page_of(blk + (STAGES + 1) * WARPS);
        }
    }
    if (!alive) {
        // wait (bounded) for the copies still on their way before the ring takes the states
        for (int s2 = 0; s2 < STAGES; ++s2) {
            const int i2 = it + s2, blk = my_lo + warp + i2 * WARPS;
            if (blk >= my_hi) break;
            for (uint32_t i = 0; i < WAIT_LIMIT; ++i)
                if (mbar_try_wait(bar0 + (i2 % STAGES) * 8, (i2 / STAGES) & 1)) break;
        }
    }
    __syncwarp();

    // ------------------------------------------------- the warps' states, then the cluster's
    float* mine = reinterpret_cast<float*>(smem + warp * STAGES * L::STAGE);
#pragma unroll
    for (int r = 0; r < RH; ++r) {
        float sum = l[r];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        float* st = mine + (n + 8 * r) * PART;
        if (j == 0) {
            st[DP] = m[r];
            st[DP + 1] = sum;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float y = mid[g][r];
            y += __shfl_xor_sync(0xffffffffu, y, 1);
            y += __shfl_xor_sync(0xffffffffu, y, 2);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int col = 2 * j + e;
                    st[g * 32 + 8 * (col & 3) + 4 * (col >> 2) + i] = o[g][i][2 * r + e] + y;
                }
        }
    }
    __syncthreads();
    // (column by column: a thread owns its columns of every warp's state, the rows' maxima and sums are left alone)
    for (int e = threadIdx.x; e < rows * DP; e += THREADS) {
        const int row = e / DP, ch = e - row * DP;
        float top = -INFINITY, x = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
            top = fmaxf(top, reinterpret_cast<const float*>(smem + w * STAGES * L::STAGE)[row * PART + DP]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float* st = reinterpret_cast<const float*>(smem + w * STAGES * L::STAGE) + row * PART;
            const float f = st[DP] == -INFINITY ? 0.0f : exp2_fast(st[DP] - top);
            x += f * st[ch];
        }
        reinterpret_cast<float*>(smem)[row * PART + ch] = x;
    }
    __syncthreads();
    if (threadIdx.x < rows) {
        const int row = threadIdx.x;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
            top = fmaxf(top, reinterpret_cast<const float*>(smem + w * STAGES * L::STAGE)[row * PART + DP]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float* st = reinterpret_cast<const float*>(smem + w * STAGES * L::STAGE) + row * PART;
            sum += (st[DP] == -INFINITY ? 0.0f : exp2_fast(st[DP] - top)) * st[DP + 1];
        }
        float* st = reinterpret_cast<float*>(smem) + row * PART;
        st[DP] = top;
        st[DP + 1] = sum;
    }
    if (p.parts > 1)
        cluster_sync_all();
    else
        __syncthreads();
    const uint32_t state = smem_u32(smem);
    for (int e = rank * THREADS + threadIdx.x; e < rows * DP; e += THREADS * p.parts) {
        const int row = e / DP, ch = e - row * DP;
        float x, sum;
        if (p.parts == 1) {
            const float* st = reinterpret_cast<const float*>(smem) + row * PART;
            x = st[ch];
            sum = st[DP + 1];
        } else {
            float top = -INFINITY;
            x = sum = 0.0f;
            for (int z = 0; z < p.parts; ++z) top = fmaxf(top, lds_cluster(cluster_addr(state + (row * PART + DP) * 4, z)));
            for (int z = 0; z < p.parts; ++z) {
                const uint32_t at = cluster_addr(state + row * PART * 4, z);
                const float mz = lds_cluster(at + DP * 4);
                const float f = mz == -INFINITY ? 0.0f : exp2_fast(mz - top);
                x += f * lds_cluster(at + ch * 4);
                sum += f * lds_cluster(at + (DP + 1) * 4);
            }
        }
        if (ch < p.head_dim) {
            const int at = first + row, tk = at / p.hpg, h = hk * p.hpg + at - tk * p.hpg;
            reinterpret_cast<T*>(p.out)[(long)(row0 + tk) * p.out_stride + (long)h * p.head_dim + ch] =
                prb_from_float<T>(sum > 0.0f ? x / sum : 0.0f);
        }
    }
    if (p.parts > 1) cluster_sync_all();                       // nobody leaves while its state may be read
}

template <int NG, bool LOW, typename T> int launch_one(const Args& p, cudaStream_t stream) {
    using L = Layout<NG>;
    constexpr int bytes = L::RING + L::BARS + 16;
    cudaError_t e = prb_allow_shared<attention_4bit_kernel<NG, LOW, T>>(bytes);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long)p.n_tiles * p.kv_heads * p.subs * p.parts));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.parts;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = prb_small_ctas_early() && prb_pdl_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, attention_4bit_kernel<NG, LOW, T>, p);
    return e == cudaSuccess ? 0 : (int)e;
}
}  // namespace attn4
