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
// as probabilities are rounded before any such product); p * middle is summed in 32 bits, since a group's middle may be many
// of its steps.  float32 queries, and then p * step, go as the sum of
// three bfloat16 numbers (24 bits), which makes three products of 32-bit exactness.
//
// Keys and values are the left operand (16 keys x 16 channels, 16 channels x 16 keys), queries and probabilities the
// right one (8 rows a product): one decoded token with a key/value head of its own wastes 7 of 8 columns rather than
// 15 of 16 rows, a thread looks after the steps and middles of 2 keys in 16 rather than 4, and half as many products do.  The
// scores' accumulator has keys along lanes where the probabilities' operand has rows there: the rounded numbers change
// lanes by shuffles (as_operand).
//
// What bounds it: the instructions that turn words of codes into operands and scale them (some 880 a stage of 64 keys of 64
// channels, issued in about half of the cycles: too few warps to cover their latencies, and units of unequal length in
// little more than one round of CTAs); then the bytes of the cache.
// 64 tokens at contexts of 500 to 1,000 of 25 heads of 64 (96 MB) take 41.2 us, 2.3 TB/s; 8 at 16,000 to 32,749 of 8 x 128
// with four rows a key/value head (240 MB) 74.6 us, 3.2 TB/s; one at 1,000 of 12 heads 6.8 us, a chain of look-ups, two
// stages and the parts' meeting.
// With bfloat16 queries the 8 stays in the codes of the keys (128 + c is what the bits of a code make without an
// addition) and goes with the middle: q . (128 + c) is off by 2^-24 of 136 sums of |q|, which is nothing there.
//
// One CTA takes up to 8 QN rows (a row is a token and one of the heads that share keys and values) of one tile for one
// key/value head, or one of the parts of their keys; the parts are a cluster, whose CTAs meet through distributed
// shared memory, so there is no workspace and no counter, and parts are added in the keys' order whatever came first.
// Each of its warps takes every nth stage of SK keys and keeps two stages of its own in flight (bulk copies, no
// multicast, of whole tiles where a page is a stage).  Nothing is shared between warps until the end.
#pragma once
#include <type_traits>

#include "cache4.cuh"
#include "tcgen05.cuh"

namespace attn4 {
using namespace tc5;

constexpr int MAX_WARPS = 4;
constexpr int STAGES = 2;                  // ring buffers of a warp
constexpr int MAX_PARTS = 8;               // CTAs of a cluster (portable)

// Keys of a stage: 64, or 32 where a thread's scores and results would not fit the registers.  Longer stages and more
// registers measured better than more warps: 8 x 32,749 positions of 8 x 128 88.9 us with stages of 32 keys and four CTAs an
// SM, 74.7 with 64 and two; 64 tokens at 1,000 of 25 heads of 64 41 with 64, 50 with 32.
__host__ __device__ constexpr int stage_keys(int ng, int qn, bool wide) {
    return (ng <= 2 && qn <= 2) || (qn == 1 && !wide) ? 64 : 32;
}

// CTAs of four warps that an SM takes (by their registers).
__host__ __device__ constexpr int ctas_of(int ng, int qn, bool wide) { return qn > 1 ? 2 : ng > 2 ? (wide ? 3 : 2) : 4; }

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
    int n_tiles, tile_most, subs, parts, warps;
    int heads, kv_heads, hpg;              // hpg: query heads per key/value head
    int head_dim, page_size, piece;        // piece: keys that lie together in a page and in a stage
    int max_pages, num_pages;
    int tile_bytes;
    float scale;
    int window;
    uint32_t magic;                        // 0x43004300 (see code_pair)
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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from nothing: d = a b.
__device__ __forceinline__ void mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// 16 x 8 x 8
__device__ __forceinline__ void mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ void mma8_0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0), "f"(0.0f));
}
// Codes i and i + 4 of a word as two bfloat16 numbers: 0x4300 | c is 128 + c; less 136 if CENTRED.
// `magic` comes from the launch: of two constants the compiler keeps neither in a register and spends an instruction more
// on every pair, an eighth of the kernel's.
template <bool CENTRED> __device__ __forceinline__ uint32_t code_pair(uint32_t word, int i, uint32_t magic) {
    const uint32_t u = ((word >> (4 * i)) & 0x000f000fu) | magic;
    if (!CENTRED) return u;
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

// Rows' numbers of keys n and n + 8 (lane 4 n + j: rows 2 j and 2 j + 1, or row j where EN is 1), rounded, as the right
// operand of a product over 16 keys: columns are rows, and its reduction's places 2 j, 2 j + 1 are keys j, j + 8, its
// places 2 j + 8, 2 j + 9 keys j + 4, j + 12, so that one pair moves at a time and nothing is put together again.
// (movmatrix would do it in the keys' own order, but is made of a dozen instructions here.)
template <int EN, int PIECES>
__device__ __forceinline__ void as_operand(const float (&x)[2 * EN], int lane, uint32_t (&b0)[PIECES], uint32_t (&b1)[PIECES]) {
    const int from = (lane & 3) * 4 + (lane >> 3);
    uint32_t even[PIECES];
    split2<PIECES>(x[0], x[EN], even);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        b0[i] = __shfl_sync(0xffffffffu, even[i], from);
        b1[i] = __shfl_sync(0xffffffffu, even[i], from + 16);
    }
    if (EN == 2) {
        uint32_t odd[PIECES];
        split2<PIECES>(x[1 % (2 * EN)], x[3 % (2 * EN)], odd);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const uint32_t o0 = __shfl_sync(0xffffffffu, odd[i], from), o1 = __shfl_sync(0xffffffffu, odd[i], from + 16);
            if (lane & 4) {
                b0[i] = o0;
                b1[i] = o1;
            }
        }
    }
}
// The (step, middle) pairs of a key's groups.
template <int NG> __device__ __forceinline__ void load_params(const uint8_t* p, uint32_t (&out)[NG]) {
    if (NG == 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        out[0] = w.x; out[1 % NG] = w.y; out[2 % NG] = w.z; out[3 % NG] = w.w;
    } else if (NG == 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        out[0] = w.x; out[1 % NG] = w.y;
    } else {
#pragma unroll
        for (int g = 0; g < NG; ++g) out[g] = reinterpret_cast<const uint32_t*>(p)[g];
    }
}
template <int NG, int QN, int EN, typename T> struct Layout {
    static constexpr int SK = stage_keys(NG, QN, sizeof(T) == 4), ROWS = EN == 1 ? 4 : 8 * QN;
    static constexpr int DP = NG * 32, PART = DP + 2;         // floats a row of a partial state: values, maximum, sum
    static constexpr int KIND = SK * (16 * NG + 4 * NG);      // most bytes of a stage's keys (and of its values)
    static constexpr int STAGE = 2 * KIND;
    // a warp's ring, which takes its state in the end
    static constexpr int STATE = (ROWS * PART * 4 + 15) / 16 * 16;
    static constexpr int WARP = STAGES * STAGE > STATE ? STAGES * STAGE : STATE;
    static constexpr int bytes(int warps) { return warps * (WARP + STAGES * 8) + 16; }
};

// QN: products' columns of 8 rows.  EN == 1 (QN is 1): up to 4 rows, in the columns 0, 2, 4 and 6, so that a thread has one
// row's scores rather than two.  FAST: the head size is 32 NG and a stage lies in one page, so that every offset is known
// here.
template <int NG, int QN, int EN, typename T, bool FAST>
__global__ void __launch_bounds__(MAX_WARPS * 32, ctas_of(NG, QN, sizeof(T) == 4))
attention_4bit_kernel(const Args p) {
    using L = Layout<NG, QN, EN, T>;
    constexpr int SK = L::SK, ROWS = L::ROWS, NC = SK / 16, DP = L::DP, PART = L::PART;
    constexpr int PIECES = sizeof(T) == 4 ? 3 : 1;
    constexpr bool EXACT = PIECES == 3;                       // codes less 8 in the keys' products too
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.warps * L::WARP);
    volatile int* failed = reinterpret_cast<volatile int*>(bars + p.warps * STAGES);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = lane >> 2, j = lane & 3;
    const int threads = p.warps * 32;
    prb_grid_launch_dependents();
    if (threadIdx.x < p.warps * STAGES) mbar_init(smem_u32(&bars[threadIdx.x]), 1);
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

    // ------------------------------------------------------------------------ stages
    const uint32_t ring = smem_u32(smem) + warp * L::WARP;
    const uint8_t* ring_p = smem + warp * L::WARP;
    const uint32_t bar0 = smem_u32(&bars[warp * STAGES]);
    const int head_dim = FAST ? DP : p.head_dim;
    const int piece = FAST ? SK : p.piece;                    // 16, 32 or 64
    const int pieces = SK / piece, piece_log = __popc(piece - 1);
    const int piece_bytes = piece * (head_dim / 2 + 4 * NG);
    const int codes_of_page = p.page_size * (head_dim / 2);
    // Lane i looks after piece i of a stage: its page, ahead of time, and its copies.
    const int per_page = FAST ? p.page_size / SK : 1;         // stages of a page
    auto page_of = [&](int blk) -> int {
        if (FAST) return blk < my_hi ? table[per_page == 1 ? blk : blk / per_page] : -2;
        const int key = blk * SK + lane * piece;
        if (blk >= my_hi || lane >= pieces || key > pos_hi || key + piece <= key_lo) return -2;    // nothing to fetch
        return table[key / p.page_size];
    };
    // (FAST: lane i has copy i of a stage, keys' and values' in turn: a page's tile, or its groups' codes and its pairs)
    const int copy = lane >> 1;
    const bool copies = FAST && copy < (per_page == 1 ? 1 : NG + 1);
    const uint8_t* copy_from = (lane & 1 ? p.v_tiles : p.k_tiles) + (size_t)hk * p.tile_bytes +
                               (copy < NG ? copy * p.page_size * 16 : codes_of_page);
    const uint32_t copy_bytes = per_page == 1 ? L::KIND : SK * (copy < NG ? 16 : NG * 4);
    const uint32_t copy_to = ring + (lane & 1) * L::KIND + copy * SK * 16;
    const size_t page_stride = (size_t)p.kv_heads * p.tile_bytes;
    auto request = [&](int blk, int st, int page) {
        if (FAST) {
            const uint32_t bar = bar0 + st * 8;
            const bool fine = page >= 0 && page < p.num_pages;
            if (lane == 0) {
                if (!fine) prb_set_status(p.status, PRB_S_PAGE_RANGE, row0, blk * SK, page);
                mbar_expect_tx(bar, fine ? 2 * L::KIND : 0);
            }
            __syncwarp();
            // (a page that is none: recorded, the stage keeps what it held, and the tile's result is not to be used)
            if (copies && fine) {
                const int at = per_page == 1 ? 0 : (blk % per_page) * SK * (copy < NG ? 16 : NG * 4);
                bulk_load(copy_to + st * L::STAGE, copy_from + (size_t)page * page_stride + at, copy_bytes, bar);
            }
            return;
        }
        bool fetch = page != -2;
        if (fetch && (page < 0 || page >= p.num_pages)) {
            prb_set_status(p.status, PRB_S_PAGE_RANGE, row0, blk * SK + lane * piece, page);
            fetch = false;
        }
        const unsigned who = __ballot_sync(0xffffffffu, fetch);
        const uint32_t bar = bar0 + st * 8;
        if (lane == 0) mbar_expect_tx(bar, (uint32_t)(__popc(who) * 2 * piece_bytes));
        __syncwarp();
        if (!fetch) return;
        const int at = (blk * SK + lane * piece) % p.page_size;
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            const uint8_t* src = (kind ? p.v_tiles : p.k_tiles) + ((size_t)page * p.kv_heads + hk) * (size_t)p.tile_bytes;
            uint32_t dst = ring + st * L::STAGE + kind * L::KIND + lane * piece_bytes;
            if (piece == p.page_size) {
                bulk_load(dst, src, piece_bytes, bar);
            } else {
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const int row = min(16, (head_dim - g * 32) / 2);
                    bulk_load(dst, src + g * p.page_size * 16 + at * row, piece * row, bar);
                    dst += piece * row;
                }
                bulk_load(dst, src + codes_of_page + at * NG * 4, piece * NG * 4, bar);
            }
        }
    };
#pragma unroll
    for (int st = 0; st < STAGES; ++st) {
        const int blk = my_lo + warp + st * p.warps;
        if (blk < my_hi) request(blk, st, page_of(blk));
    }
    int ahead = page_of(my_lo + warp + STAGES * p.warps);

    // ---------------------------------------------------------------------- queries
    // Channel order of the reduction: thread j of a quad has channels 8 j + (i, i + 4), the codes that one shift and
    // one mask take from word j.
    uint32_t qb[QN][NG][2][PIECES][2];                        // [rows][group][half of the reduction][piece][operand]
    // What a key's steps and middles are multiplied by in a score, as three bfloat16 numbers each: less 136 sums of q
    // (where the codes are 128 + c) and the sum of q, of group j.
    uint32_t qp[QN][3];
    int pos[QN][EN];
#pragma unroll
    for (int z = 0; z < QN; ++z) {
        float mine = 0.0f;
        // (column n of the products)
        const int row = EN == 1 ? n >> 1 : n + 8 * z, at = first + min(row, rows - 1);
        const bool used = row < rows && (EN == 2 || (n & 1) == 0);
        const int tk = at / p.hpg, h = hk * p.hpg + at - tk * p.hpg;
        const int here = pos0 + tk;
#pragma unroll
        for (int e = 0; e < EN; ++e) pos[z][e] = __shfl_sync(0xffffffffu, here, (2 * j + e) * 4);
        const T* src = reinterpret_cast<const T*>(p.q) + (long)(row0 + tk) * p.q_stride + (long)h * head_dim;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int c0 = g * 32 + j * 8;
            float x[8];
            if (used && c0 < head_dim) {
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
            if (j == g) mine = sum;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w[PIECES];
                split2<PIECES>(x[i], x[i + 4], w);
#pragma unroll
                for (int y = 0; y < PIECES; ++y) qb[z][g][i >> 1][y][i & 1] = w[y];
            }
        }
        split2<3>(EXACT ? 0.0f : -136.0f * mine, mine, qp[z]);
    }

    // results [rows][group][16 of its channels]: channels (2 i, 2 i + 1 of the thread's four) x rows (2 j, 2 j + 1); sums of
    // p * middle over the lane's keys, of rows 2 j, 2 j + 1
    float o[QN][NG][2][4], mid[QN][EN][NG];
    float m[QN][EN], l[QN][EN];
#pragma unroll
    for (int z = 0; z < QN; ++z) {
#pragma unroll
        for (int e = 0; e < EN; ++e) {
            m[z][e] = -INFINITY;
            l[z][e] = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) mid[z][e][g] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int g = 0; g < NG; ++g) o[z][g][0][i] = o[z][g][1][i] = 0.0f;
    }
    const float sl2 = p.scale * 1.4426950408889634f;          // scores are handled in log2 units
    // (the short last group's rows are 8 bytes apart; its words 2 and 3 do not exist: words 0 and 1 stand in, against
    // queries of zero and for channels that are not stored)
    const bool short_last = !FAST && head_dim % 32 != 0;

    const uint32_t magic = p.magic;
    // A stage's keys and values: scores, exponentials, results.
    auto work = [&](int st, int key0, auto masked_t) {
        constexpr bool masked = decltype(masked_t)::value;
        const uint8_t* ks = ring_p + st * L::STAGE;
        const uint8_t* vs = ks + L::KIND;
        // ---- scores of keys n and n + 8 of every 16
        float s[NC][QN][2 * EN];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int pc = FAST ? 0 : (c * 16) >> piece_log, in = c * 16 - pc * piece;
            const uint8_t* base = ks + pc * piece_bytes;
            const uint8_t* par = base + piece * (head_dim / 2) + (in + n) * NG * 4;
            uint32_t pr[2][NG];
            load_params<NG>(par, pr[0]);
            load_params<NG>(par + 8 * NG * 4, pr[1]);
            // steps and middles against the sums of q: numbers 2 j, 2 j + 1 of the reduction are group j's
            const int jg = NG == 4 ? j : min(j, NG - 1);
            const uint32_t p0 = *reinterpret_cast<const uint32_t*>(par + jg * 4);
            const uint32_t p1 = *reinterpret_cast<const uint32_t*>(par + 8 * NG * 4 + jg * 4);
            float sum[QN][4];
#pragma unroll
            for (int z = 0; z < QN; ++z) {
                mma8_0(sum[z], p0, p1, qp[z][2]);
                mma8(sum[z], p0, p1, qp[z][1]);
                mma8(sum[z], p0, p1, qp[z][0]);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const bool sh = g == NG - 1 && short_last;
                const uint8_t* word = base + g * piece * 16 + (sh ? (in + n) * 8 + (j & 1) * 4 : (in + n) * 16 + j * 4);
                const uint32_t w0 = *reinterpret_cast<const uint32_t*>(word);
                const uint32_t w1 = *reinterpret_cast<const uint32_t*>(word + (sh ? 64 : 128));
                uint32_t a[4][2];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i][0] = code_pair<EXACT>(w0, i, magic);
                    a[i][1] = code_pair<EXACT>(w1, i, magic);
                }
                const float step0 = __uint_as_float(pr[0][g] << 16), step1 = __uint_as_float(pr[1][g] << 16);
#pragma unroll
                for (int z = 0; z < QN; ++z) {
                    float acc[4];
#pragma unroll
                    for (int y = PIECES - 1; y >= 0; --y) {
                        if (y == PIECES - 1)
                            mma0(acc, a[0][0], a[0][1], a[1][0], a[1][1], qb[z][g][0][y][0], qb[z][g][0][y][1]);
                        else
                            mma(acc, a[0][0], a[0][1], a[1][0], a[1][1], qb[z][g][0][y][0], qb[z][g][0][y][1]);
                        mma(acc, a[2][0], a[2][1], a[3][0], a[3][1], qb[z][g][1][y][0], qb[z][g][1][y][1]);
                    }
#pragma unroll
                    for (int e = 0; e < EN; ++e) {
                        sum[z][e] = fmaf(step0, acc[e], sum[z][e]);
                        sum[z][e + 2] = fmaf(step1, acc[e + 2], sum[z][e + 2]);
                    }
                }
            }
#pragma unroll
            for (int z = 0; z < QN; ++z)
#pragma unroll
                for (int e = 0; e < EN; ++e) {
                    s[c][z][e] = sum[z][e];
                    s[c][z][e + EN] = sum[z][e + 2];
                }
        }
        // (which weights are 0 because their key is masked: a weight that is 0 because e^x has no smaller number still makes NaN
        // of a value that is none)
        uint32_t hidden = 0;
        static_assert(NC * QN * 2 * EN <= 32, "a bit a score");
        auto is_hidden = [&](int c, int z, int e) -> bool { return (hidden >> ((c * QN + z) * 2 * EN + e)) & 1u; };
        if (masked) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int z = 0; z < QN; ++z)
#pragma unroll
                    for (int e = 0; e < 2 * EN; ++e) {
                        const int key = key0 + c * 16 + n + 8 * (e / EN), at = pos[z][e % EN];
                        if (key > at || (p.window > 0 && key <= at - p.window)) {
                            s[c][z][e] = -INFINITY;
                            hidden |= 1u << ((c * QN + z) * 2 * EN + e);
                        }
                    }
        }
        // ---- maximum, exponentials
        float alpha[QN][EN];
        bool moved = false;
#pragma unroll
        for (int z = 0; z < QN; ++z)
#pragma unroll
            for (int e = 0; e < EN; ++e) {
                float top = -INFINITY;
#pragma unroll
                for (int c = 0; c < NC; ++c) top = fmaxf(top, fmaxf(s[c][z][e], s[c][z][e + EN]));
#pragma unroll
                for (int o2 = 4; o2 < 32; o2 <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o2));
                const float now = fmaxf(m[z][e], top * sl2);
                const float ref = now == -INFINITY ? 0.0f : now;
                alpha[z][e] = exp2_fast(m[z][e] - ref);       // (0 while nothing was seen)
                moved = moved || alpha[z][e] != 1.0f;
                m[z][e] = now;
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int k = e; k < 2 * EN; k += EN) {
                        s[c][z][k] = exp2_fast(fmaf(s[c][z][k], sl2, -ref));
                        sum += s[c][z][k];
                    }
                l[z][e] = fmaf(l[z][e], alpha[z][e], sum);
            }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int z = 0; z < QN; ++z)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if ((i & 1) >= EN) continue;
                    const float by = alpha[z][(i & 1) % EN];
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        if (i < 2) mid[z][i % EN][g] *= by;
                        o[z][g][0][i] *= by;
                        o[z][g][1][i] *= by;
                    }
                }
        }
        // ---- values
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int pc = FAST ? 0 : (c * 16) >> piece_log, in = c * 16 - pc * piece;
            const uint8_t* base = vs + pc * piece_bytes;
            const uint8_t* par = base + piece * (head_dim / 2) + in * NG * 4;
            uint32_t pr[2][NG];
            load_params<NG>(par + n * NG * 4, pr[0]);
            load_params<NG>(par + (n + 8) * NG * 4, pr[1]);
            // p * middle, in 32 bits: a lane's keys by themselves, all lanes' in the end.  (A masked key's middle may be
            // anything, NaN too.)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float middle0 = __uint_as_float(pr[0][g] & 0xffff0000u), middle1 = __uint_as_float(pr[1][g] & 0xffff0000u);
#pragma unroll
                for (int z = 0; z < QN; ++z)
#pragma unroll
                    for (int e = 0; e < EN; ++e) {
                        if (!masked || !is_hidden(c, z, e)) mid[z][e][g] = fmaf(s[c][z][e], middle0, mid[z][e][g]);
                        if (!masked || !is_hidden(c, z, e + EN)) mid[z][e][g] = fmaf(s[c][z][e + EN], middle1, mid[z][e][g]);
                    }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const bool sh = g == NG - 1 && short_last;
                const uint8_t* col = base + g * piece * 16 + (sh ? (n & 1) * 4 : (n & 3) * 4) + (n >> 2) * 2;
                auto half = [&](int key) -> uint32_t {
                    return *reinterpret_cast<const uint16_t*>(col + (in + key) * (sh ? 8 : 16));
                };
                const uint32_t u = half(j) | (half(j + 8) << 16);
                const uint32_t v = half(j + 4) | (half(j + 12) << 16);
                uint32_t a[4][2];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i][0] = code_pair<true>(u, i, magic);
                    a[i][1] = code_pair<true>(v, i, magic);
                }
                const float step0 = __uint_as_float(pr[0][g] << 16), step1 = __uint_as_float(pr[1][g] << 16);
#pragma unroll
                for (int z = 0; z < QN; ++z) {
                    float x[2 * EN];
#pragma unroll
                    for (int e = 0; e < EN; ++e) {
                        x[e] = s[c][z][e] * step0;
                        x[e + EN] = s[c][z][e + EN] * step1;
                        if (masked) {
                            if (is_hidden(c, z, e)) x[e] = 0.0f;
                            if (is_hidden(c, z, e + EN)) x[e + EN] = 0.0f;
                        }
                    }
                    uint32_t b0[PIECES], b1[PIECES];
                    as_operand<EN, PIECES>(x, lane, b0, b1);
                    if (EXACT) {
                        // The matrix units cut what a sum in 32 bits does not hold instead of rounding it, and thousands
                        // of keys make that a drift (1.7e-6 at contexts of some 10,000): 16 keys at a time there, the
                        // rest in sums that round.
                        float part[2][4];
                        mma0(part[0], a[0][0], a[1][0], a[0][1], a[1][1], b0[PIECES - 1], b1[PIECES - 1]);
                        mma0(part[1], a[2][0], a[3][0], a[2][1], a[3][1], b0[PIECES - 1], b1[PIECES - 1]);
#pragma unroll
                        for (int k = PIECES - 2; k >= 0; --k) {
                            mma(part[0], a[0][0], a[1][0], a[0][1], a[1][1], b0[k], b1[k]);
                            mma(part[1], a[2][0], a[3][0], a[2][1], a[3][1], b0[k], b1[k]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if ((e & 1) >= EN) continue;
                            o[z][g][0][e] += part[0][e];
                            o[z][g][1][e] += part[1][e];
                        }
                    } else {
                        mma(o[z][g][0], a[0][0], a[1][0], a[0][1], a[1][1], b0[0], b1[0]);
                        mma(o[z][g][1], a[2][0], a[3][0], a[2][1], a[3][1], b0[0], b1[0]);
                    }
                }
            }
        }
    };

    bool alive = true;
    int it = 0;
    for (int blk = my_lo + warp; blk < my_hi; blk += p.warps, ++it) {
        const int st = it % STAGES;
        alive = mbar_wait_warp(bar0 + st * 8, (it / STAGES) & 1, failed);
        if (!alive) {
            if (lane == 0) prb_set_status(p.status, PRB_S_WAIT_TIMEOUT, 41, blockIdx.x, blk);
            break;
        }
        // (two copies of the work, since a stage without a masked key should not carry what one needs)
        const int key0 = blk * SK;
        if (key0 + SK - 1 > pos_lo || (p.window > 0 && key0 <= pos_hi - p.window))
            work(st, key0, std::true_type());
        else
            work(st, key0, std::false_type());
        __syncwarp();                                          // every lane has read the stage
        if (blk + STAGES * p.warps < my_hi) {
            request(blk + STAGES * p.warps, st, ahead);
            ahead = page_of(blk + (STAGES + 1) * p.warps);
        }
    }
    if (!alive) {
        // wait (bounded) for the copies still on their way before the ring takes the states
        for (int s2 = 0; s2 < STAGES; ++s2) {
            const int i2 = it + s2, blk = my_lo + warp + i2 * p.warps;
            if (blk >= my_hi) break;
            for (uint32_t i = 0; i < WAIT_LIMIT; ++i)
                if (mbar_try_wait(bar0 + (i2 % STAGES) * 8, (i2 / STAGES) & 1)) break;
        }
    }
    __syncwarp();

    // ------------------------------------------------- the warps' states, then the cluster's
    float* mine = reinterpret_cast<float*>(smem + warp * L::WARP);
#pragma unroll
    for (int z = 0; z < QN; ++z)
#pragma unroll
        for (int e = 0; e < EN; ++e) {
            float sum = l[z][e];
#pragma unroll
            for (int o2 = 4; o2 < 32; o2 <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o2);
            const int row = EN == 1 ? j : 8 * z + 2 * j + e;
            float* st = mine + row * PART;
            if (n == 0) {
                st[DP] = m[z][e];
                st[DP + 1] = sum;
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float y = mid[z][e][g];
#pragma unroll
                for (int o2 = 4; o2 < 32; o2 <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o2);
                float* at = st + g * 32 + 8 * (n & 3) + 4 * (n >> 2);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    at[2 * i] = o[z][g][i][e] + y;
                    at[2 * i + 1] = o[z][g][i][e + 2] + y;
                }
            }
        }
    __syncthreads();
    if (p.warps > 1) {
        // (a thread owns its column of every warp's state; the maxima and sums are left alone until all have read them)
        for (int e = threadIdx.x; e < rows * DP; e += threads) {
            const int row = e / DP, ch = e - row * DP;
            float top = -INFINITY, x = 0.0f;
            for (int w = 0; w < p.warps; ++w)
                top = fmaxf(top, reinterpret_cast<const float*>(smem + w * L::WARP)[row * PART + DP]);
            for (int w = 0; w < p.warps; ++w) {
                const float* st = reinterpret_cast<const float*>(smem + w * L::WARP) + row * PART;
                x += (st[DP] == -INFINITY ? 0.0f : exp2_fast(st[DP] - top)) * st[ch];
            }
            reinterpret_cast<float*>(smem)[row * PART + ch] = x;
        }
        __syncthreads();
        if (threadIdx.x < rows) {
            const int row = threadIdx.x;
            float top = -INFINITY, sum = 0.0f;
            for (int w = 0; w < p.warps; ++w)
                top = fmaxf(top, reinterpret_cast<const float*>(smem + w * L::WARP)[row * PART + DP]);
            for (int w = 0; w < p.warps; ++w) {
                const float* st = reinterpret_cast<const float*>(smem + w * L::WARP) + row * PART;
                sum += (st[DP] == -INFINITY ? 0.0f : exp2_fast(st[DP] - top)) * st[DP + 1];
            }
            float* st = reinterpret_cast<float*>(smem) + row * PART;
            st[DP] = top;
            st[DP + 1] = sum;
        }
    }
    if (p.parts > 1)
        cluster_sync_all();
    else
        __syncthreads();
    const uint32_t state = smem_u32(smem);
    for (int e = rank * threads + threadIdx.x; e < rows * DP; e += threads * p.parts) {
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
        if (ch < head_dim) {
            const int at = first + row, tk = at / p.hpg, h = hk * p.hpg + at - tk * p.hpg;
            reinterpret_cast<T*>(p.out)[(long)(row0 + tk) * p.out_stride + (long)h * head_dim + ch] =
                prb_from_float<T>(sum > 0.0f || sum != sum ? x / sum : 0.0f);      // (a NaN goes on)
        }
    }
    if (p.parts > 1) cluster_sync_all();                       // nobody leaves while its state may be read
}

template <int NG, int QN, int EN, typename T, bool FAST> int launch_one(const Args& p, cudaStream_t stream) {
    using L = Layout<NG, QN, EN, T>;
    cudaError_t e = prb_allow_shared<attention_4bit_kernel<NG, QN, EN, T, FAST>>(L::bytes(MAX_WARPS));
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long)p.n_tiles * p.kv_heads * p.subs * p.parts));
    cfg.blockDim = dim3(p.warps * 32);
    cfg.dynamicSmemBytes = L::bytes(p.warps);
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
    e = cudaLaunchKernelEx(&cfg, attention_4bit_kernel<NG, QN, EN, T, FAST>, p);
    return e == cudaSuccess ? 0 : (int)e;
}

// `p` but for subs, parts, warps and piece is set; rows: the most rows of a tile.
template <int NG, int QN, int EN, typename T> int launch_by(Args p, long rows, int max_context, int parts, cudaStream_t stream) {
    constexpr int sk = stage_keys(NG, QN, sizeof(T) == 4);
    p.piece = p.page_size % sk == 0 ? sk : p.page_size % 32 == 0 ? 32 : 16;
    if (sk % p.page_size == 0) p.piece = p.page_size;
    constexpr int most = Layout<NG, QN, EN, T>::ROWS;
    const long subs = (rows + most - 1) / most, units = (long)p.n_tiles * p.kv_heads * subs;
    if (units > 0x7fffffffL / MAX_PARTS) return PRB_E_SIZE;
    p.subs = (int)subs;
    // Four warps a CTA; two once the units alone fill the SMs with such CTAs: a warp then has twice the stages to
    // one set-up and half as many states to merge.  64 tokens at 1,000 of 12 heads (768 units) 26.7 us with four, 22.2 with
    // two; at 300 of 16 heads (1,024) 15.2 and 13.0; 24 x 5 tokens of 16 heads (384) 13.9 and 19.2; float32 texts (more
    // instructions a stage) 32.4 and 41.8.
    const long slots = (long)ctas_of(NG, QN, sizeof(T) == 4) * prb_sm_count();
    p.warps = QN == 1 && sizeof(T) == 2 && units > slots ? 2 : MAX_WARPS;
    // Parts of a unit's keys while all CTAs still run side by side, each with a stage a warp at least.  (The longest
    // request's: max_context, or what a window and the tile's own tokens span.)
    const int reach = p.window > 0 ? min((long)max_context, (long)p.window + p.tile_most + sk) : max_context;
    const int stages = (reach + sk - 1) / sk + (p.window > 0 ? 1 : 0);   // (a window need not begin with a stage)
    p.parts = 1;
    while (p.parts < MAX_PARTS && units * p.parts * 2 <= slots && stages >= p.parts * 2 * p.warps) p.parts *= 2;
    if (parts > 0) p.parts = parts;
    if (p.piece == sk && p.head_dim == 32 * NG) return launch_one<NG, QN, EN, T, true>(p, stream);
    return launch_one<NG, QN, EN, T, false>(p, stream);
}
}  // namespace attn4
