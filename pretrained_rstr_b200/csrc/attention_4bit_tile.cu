// Causal attention of prompt portions over a cache held in 4 bits (cache4.cuh) on the 5th-generation tensor cores.
// bfloat16, no window; operands are 64 or 128 channels wide, what a head size leaves of them is zero.
//
// One CTA takes up to 128 rows (tokens times the query heads of one key/value head) of a tile and walks the keys in
// blocks of 64, or one of the parts of them (parts are a cluster and meet through distributed shared memory).  Warps:
//   0      producer: bulk copies of a block's codes, steps and middles (5 KB at head size 64 for keys and values, where
//          bfloat16 is 16) into a ring of raw stages;
//   1      allocates tensor memory; one thread issues tcgen05.mma: S = Q K^T (128 x 64), O += P V;
//   2-9    softmax: two threads a row, each 32 of a block's 64 scores and half of the output's channels;
//   10-17  turn codes into operands in the swizzled layout, once for all 128 rows.
// Weights become bfloat16 (2^-8, as before any such product; their sum is of the unrounded ones), and so do values (2^-8 of
// a value, as a bfloat16 cache would hold it, on top of the cache's own rounding).  Keys
// become the sum of two bfloat16 numbers and take two products: a key's rounding moves a score by the product of the
// query's and the key's lengths times it, which at ordinary scores is several times what P's rounding costs, and the tensor
// cores wait for the softmax anyway.
//
// Measured: portions of 4 x 512 tokens at contexts of 4,000, 16 heads of 64 (16.5 GFLOP) 99.5 us, where tiles of 32 rows on
// mma.sync take 200 (and with a window of 1,000, which only they know, 115); 512 tokens at 8,000 of 32 heads over 8 x 128
// (65 GFLOP) 185 us, 350 TFLOP/s.  What bounds it: the
// instructions of softmax and conversion (5,900 a block of 64 keys, a third of them the conversion, in 70 % of the issue
// slots while a CTA pair runs), and the SMs that one tile less leaves with one CTA where others have two.  Eight warps
// convert: with four the blocks waited for them (512 tokens at 8,000: 302 us).
//
// What lies behind the tile's last position (stale pages, NaN) becomes zeros.  A key that the tile's later tokens see and
// its earlier ones do not may read back as NaN, or as more than bfloat16's largest number (3.39e38): it becomes zeros too,
// and the rows that see it are made NaN in the channels of its group at the end, since a product would spread it over all
// rows.
//
// Every wait is bounded: where one gives up the status word says so, its CTA stores nothing more, copies in flight are
// waited for, tensor memory is freed.
#include <type_traits>

#include "cache4.cuh"
#include "tcgen05.cuh"

namespace {
using namespace tc5;

constexpr int QT = 128, KB = 64;
constexpr int SOFTMAX = 8, DEQUANT = 8, WARPS = 2 + SOFTMAX + DEQUANT, THREADS = WARPS * 32;
constexpr int RAW_STAGES = 3, STAGES = 2, MAX_PARTS = 4;
constexpr int P_BYTES = QT * KB * 2;
constexpr float RESCALE_STEP = 8.0f;         // a row's reference maximum moves only by more than this (log2 units)

// ND: operands' width / 64.
template <int ND> struct Sizes {
    static constexpr int D = 64 * ND, NG = 2 * ND;
    static constexpr int RAW = KB * (D / 2 + 4 * NG);           // most bytes of a block's keys (and of its values)
    static constexpr int TILE = KB * 128;                       // 64 keys x 64 channels of bfloat16
    static constexpr int STAGE = 3 * ND * TILE;                 // keys, what their rounding left, values
    static constexpr int Q_BYTES = QT * D * 2;
    static constexpr int STATE = QT * D * 4;                    // a part's results, in the stages' place
    static_assert(STATE <= STAGES * STAGE, "a part's results fit the stages");
    static constexpr size_t SMEM = 1024 + Q_BYTES + P_BYTES + STAGES * STAGE + RAW_STAGES * 2 * RAW + 256 + 6 * QT * 4;
};

struct Params {
    __nv_bfloat16* out;
    long out_stride;
    const __nv_bfloat16* q;
    long q_stride;
    const uint8_t* k_tiles;
    const uint8_t* v_tiles;
    const int* block_table;
    const int* positions;
    const int* tile_req;
    const int* tile_row0;
    const int* tile_rows;
    const int* tile_count;
    int n_tokens, n_requests, n_tiles, subs, parts;
    int kv_heads, hpg, head_dim, page_size, max_pages, num_pages, tile_bytes;
    int piece;                              // keys that lie together in a page and in a block: 64, 32 or 16
    float scale;
    uint32_t magic;                         // 0x43004300: a constant that the compiler keeps in a register
    int* status;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 32 lanes x 16 consecutive 32-bit columns, to and from tensor memory.
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float lds_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// FULL: the head size is 64 ND and a block lies in one page, so that the layouts are known here (a tenth of the time).
template <int ND, bool FULL>
__global__ void __launch_bounds__(THREADS, ND == 1 ? 2 : 1) attention_4bit_tile_kernel(const Params p) {
    using Z = Sizes<ND>;
    constexpr int D = Z::D, NG = Z::NG, RAW = Z::RAW, TILE = Z::TILE, STAGE = Z::STAGE;
    constexpr uint32_t TMEM_COLS = 256, O_COL = 2 * KB;         // two score buffers, then the results
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_s = smem;
    uint8_t* p_s = smem + Z::Q_BYTES;
    uint8_t* ring = p_s + P_BYTES;
    uint8_t* raw = ring + STAGES * STAGE;
    uint64_t* bars = reinterpret_cast<uint64_t*>(raw + RAW_STAGES * 2 * RAW);
    uint64_t* raw_full = bars;                   // [RAW_STAGES] copies -> dequant
    uint64_t* raw_empty = raw_full + RAW_STAGES; // dequant -> copies
    uint64_t* k_full = raw_empty + RAW_STAGES;   // [STAGES] dequant -> MMA
    uint64_t* k_empty = k_full + STAGES;         // MMA -> dequant: a block's keys are free before its softmax begins
    uint64_t* v_full = k_empty + STAGES;
    uint64_t* v_empty = v_full + STAGES;
    uint64_t* s_full = v_empty + STAGES;         // [2] scores ready
    uint64_t* q_full = s_full + 2;
    uint64_t* p_full = q_full + 1;
    uint64_t* o_full = p_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 1);
    volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* poison = reinterpret_cast<int*>(tmem_slot + 2);        // [NG] first key whose values are no numbers
    float* xmax = reinterpret_cast<float*>(bars + 32);          // [2 blocks][2 halves][QT]
    float* state_m = xmax + 4 * QT;                             // [QT] maximum and sum of a part's rows
    float* state_l = state_m + QT;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    prb_grid_launch_dependents();
    prb_grid_wait();

    // (whole clusters leave: their unit is one)
    const int unit = blockIdx.x / p.parts, rank = blockIdx.x - unit * p.parts;
    const int per = p.kv_heads * p.subs;
    const int tile = unit / per;
    const int hk = (unit - tile * per) / p.subs, sub = unit - tile * per - hk * p.subs;
    const int n_tiles = p.tile_count != nullptr ? min(*p.tile_count, p.n_tiles) : p.n_tiles;
    if (tile >= n_tiles) return;
    const int req = p.tile_req[tile], row0 = p.tile_row0[tile], tokens = p.tile_rows[tile];
    const int first = sub * QT;
    if (tokens <= 0 || first >= tokens * p.hpg) return;
    const bool placed = req >= 0 && req < p.n_requests && row0 >= 0 && tokens <= p.n_tokens && row0 <= p.n_tokens - tokens;
    const int pos0 = placed ? p.positions[row0] : -1;
    if (pos0 < 0 || pos0 > p.max_pages * p.page_size - tokens || tokens * p.hpg > p.subs * QT) {
        if (threadIdx.x == 0 && rank == 0) prb_set_status(p.status, PRB_S_POSITION_RANGE, row0, pos0, tokens);
        return;
    }
    const int rows = min(QT, tokens * p.hpg - first);
    const int pos_lo = pos0 + first / p.hpg, pos_hi = pos0 + (first + rows - 1) / p.hpg;
    const int all_blocks = pos_hi / KB + 1;
    const int blk_lo = (int)((long)all_blocks * rank / p.parts);
    const int n_blocks = (int)((long)all_blocks * (rank + 1) / p.parts) - blk_lo;
    const int* table = p.block_table + (size_t)req * p.max_pages;
    const int head_dim = FULL ? D : p.head_dim, ng = FULL ? NG : cache4::groups_of(head_dim);
    const int piece = FULL ? KB : p.piece;

    if (threadIdx.x == 0) {
        for (int s = 0; s < RAW_STAGES; ++s) {
            mbar_init(smem_u32(&raw_full[s]), 1);
            mbar_init(smem_u32(&raw_empty[s]), DEQUANT);
        }
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&k_full[s]), DEQUANT);
            mbar_init(smem_u32(&k_empty[s]), 1);
            mbar_init(smem_u32(&v_full[s]), DEQUANT);
            mbar_init(smem_u32(&v_empty[s]), 1);
        }
        mbar_init(smem_u32(&s_full[0]), 1);
        mbar_init(smem_u32(&s_full[1]), 1);
        mbar_init(smem_u32(q_full), SOFTMAX);
        mbar_init(smem_u32(p_full), SOFTMAX);
        mbar_init(smem_u32(o_full), 1);
        *failed = 0;
        for (int g = 0; g < NG; ++g) poison[g] = 0x7fffffff;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    // what a softmax thread leaves for the end
    const int quarter = warp & 3, half = (warp - 2) >> 2, r = quarter * 32 + lane;
    const bool softmax = warp >= 2 && warp < 2 + SOFTMAX;
    float m_run = -INFINITY, l_all = 0.0f;
    bool ok = true;

    if (warp == 0) {
        // ------------------------------------------------------------------ producer
        // A block's bytes go where one page of 64 would have them, whatever pages they come from: lane i looks after the page
        // of piece i, copies (a group's codes, or the pairs, of keys or values of a piece) go around the lanes.
        const int pieces = KB / piece, row_bytes = head_dim / 2 + 4 * ng, codes_of_page = p.page_size * (head_dim / 2);
        const int copies = pieces * (ng + 1) * 2;
        auto page_of = [&](int blk) -> int {
            const int key = blk * KB + lane * piece;
            return lane < pieces && key <= pos_hi ? table[key / p.page_size] : -2;       // -2: nothing to fetch
        };
        int j = 0;
        int page = page_of(blk_lo);
        for (; j < n_blocks; ++j) {
            const int st = j % RAW_STAGES, key0 = (blk_lo + j) * KB;
            ok = mbar_wait_warp(smem_u32(&raw_empty[st]), ((j / RAW_STAGES) & 1) ^ 1, failed);
            if (!ok) {
                if (lane == 0) prb_set_status(p.status, PRB_S_WAIT_TIMEOUT, 43, blockIdx.x, j);
                break;
            }
            const uint32_t fb = smem_u32(&raw_full[st]);
            const bool fine = page >= 0 && page < p.num_pages;
            // (a page that is none: recorded, the stage keeps what it held, and the tile's result is not to be used)
            if (!fine && page != -2) prb_set_status(p.status, PRB_S_PAGE_RANGE, row0, key0 + lane * piece, page);
            const unsigned who = __ballot_sync(0xffffffffu, fine);
            if (lane == 0) mbar_expect_tx(fb, (uint32_t)(__popc(who) * 2 * piece * row_bytes));
            __syncwarp();
            const uint32_t dst = smem_u32(raw) + st * 2 * RAW;
            if (p.page_size == KB) {
                const int pg = __shfl_sync(0xffffffffu, page, 0);
                if (lane < 2 && (who & 1))
                    bulk_load(dst + lane * RAW,
                              (lane ? p.v_tiles : p.k_tiles) + ((size_t)pg * p.kv_heads + hk) * (size_t)p.tile_bytes,
                              KB * row_bytes, fb);
            } else {
                for (int i0 = 0; i0 < copies; i0 += 32) {
                    const int i = i0 + lane, kind = i & 1, c = (i >> 1) % (ng + 1), pc = min((i >> 1) / (ng + 1), pieces - 1);
                    const int pg = __shfl_sync(0xffffffffu, page, pc);
                    if (i < copies && ((who >> pc) & 1)) {
                        const int in = pc * piece, at = (key0 + in) % p.page_size;
                        const int row = c == ng ? 4 * ng : min(16, (head_dim - c * 32) / 2);
                        const uint8_t* src = (kind ? p.v_tiles : p.k_tiles) + ((size_t)pg * p.kv_heads + hk) * (size_t)p.tile_bytes +
                                             (c == ng ? codes_of_page : c * p.page_size * 16) + at * row;
                        bulk_load(dst + kind * RAW + (c == ng ? KB * (head_dim / 2) : c * KB * 16) + in * row, src,
                                  piece * row, fb);
                    }
                }
            }
            __syncwarp();
            if (j + 1 < n_blocks) page = page_of(blk_lo + j + 1);
        }
        // copies still on their way, whoever has given up: nobody leaves before they have landed
        for (int jj = j > RAW_STAGES ? j - RAW_STAGES : 0; jj < j; ++jj)
            for (uint32_t i = 0; i < WAIT_LIMIT; ++i)
                if (mbar_try_wait(smem_u32(&raw_full[jj % RAW_STAGES]), (jj / RAW_STAGES) & 1)) break;
        __syncwarp();
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        constexpr uint32_t idesc_s = make_idesc(QT, KB);          // queries, keys: both K-major
        constexpr uint32_t idesc_o = make_idesc_b_mn(QT, 64);     // P K-major, values MN-major
        const uint64_t p_desc = make_smem_desc(smem_u32(p_s));
        auto issue_scores = [&](int j) {
            const uint32_t stage = smem_u32(ring + (size_t)(j % STAGES) * STAGE);
            const uint32_t d = tmem_base + (uint32_t)((j & 1) * KB);
            if (elect_one()) {
#pragma unroll
                for (int part = 0; part < 2; ++part)              // what the keys' rounding left first, then the keys
#pragma unroll
                    for (int a = 0; a < ND; ++a) {
                        const uint64_t q_desc = make_smem_desc(smem_u32(q_s) + a * QT * 128);
                        const uint64_t k_desc = make_smem_desc(stage + ((1 - part) * ND + a) * TILE);
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            umma_bf16(d, q_desc + (uint64_t)(kk * 2), k_desc + (uint64_t)(kk * 2), idesc_s,
                                      part > 0 || a > 0 || kk > 0 ? 1u : 0u);
                    }
                umma_commit(smem_u32(&s_full[j & 1]));
                umma_commit(smem_u32(&k_empty[j % STAGES]));
            }
            __syncwarp();
        };
        if (n_blocks > 0) {
            ok = mbar_wait_warp(smem_u32(q_full), 0, failed);
            if (ok) ok = mbar_wait_warp(smem_u32(&k_full[0]), 0, failed);
            if (ok) {
                tcgen05_fence_after();
                issue_scores(0);
            }
            for (int j = 0; j < n_blocks && ok; ++j) {
                if (j + 1 < n_blocks) {
                    ok = mbar_wait_warp(smem_u32(&k_full[(j + 1) % STAGES]), ((j + 1) / STAGES) & 1, failed);
                    if (!ok) break;
                    tcgen05_fence_after();
                    issue_scores(j + 1);
                }
                ok = mbar_wait_warp(smem_u32(&v_full[j % STAGES]), (j / STAGES) & 1, failed);
                if (ok) ok = mbar_wait_warp(smem_u32(p_full), j & 1, failed);
                if (!ok) break;
                tcgen05_fence_after();
                const uint32_t v_addr = smem_u32(ring + (size_t)(j % STAGES) * STAGE) + 2 * ND * TILE;
                if (elect_one()) {
#pragma unroll
                    for (int a = 0; a < ND; ++a)
#pragma unroll
                        for (int kk = 0; kk < KB / 16; ++kk)      // 16 keys further: two 8-row groups of 1024 bytes
                            umma_bf16(tmem_base + O_COL + a * 64, p_desc + (uint64_t)(kk * 2),
                                      make_smem_desc(v_addr + a * TILE + kk * 2048), idesc_o, j > 0 || kk > 0 ? 1u : 0u);
                    umma_commit(smem_u32(o_full));
                    umma_commit(smem_u32(&v_empty[j % STAGES]));
                }
                __syncwarp();
            }
            if (!ok && lane == 0) prb_set_status(p.status, PRB_S_WAIT_TIMEOUT, 44, blockIdx.x, 0);
        }
    } else if (softmax) {
        // -------------------------------------------------------------------- softmax
        const int row = first + min(r, rows - 1), tk = row / p.hpg;
        const bool row_ok = r < rows;
        const int qpos = pos0 + tk;
        const float sl2 = p.scale * 1.4426950408889634f;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
        constexpr int HC = KB / 2;
        {
            // the queries, in the layout that a tile copy with the 128-byte swizzle would have made
            const __nv_bfloat16* src = p.q + (long)(row0 + tk) * p.q_stride + (long)(hk * p.hpg + row - tk * p.hpg) * head_dim;
#pragma unroll
            for (int c = 0; c < 4 * ND; ++c) {
                const int ci = half * 4 * ND + c;
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (row_ok && ci * 8 < head_dim) w = *reinterpret_cast<const uint4*>(src + ci * 8);
                st_shared_v4(smem_u32(q_s) + (ci >> 3) * QT * 128 + r * 128 + (((ci & 7) ^ (r & 7)) << 4),
                             __byte_perm(w.x, w.z, 0x5410), __byte_perm(w.x, w.z, 0x7632),
                             __byte_perm(w.y, w.w, 0x5410), __byte_perm(w.y, w.w, 0x7632));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(q_full));
        }
        float l_run = 0.0f;
        for (int j = 0; j < n_blocks; ++j) {
            // After a wait gave up the warp still walks every block, without waiting or touching tensor memory, so that
            // the barriers of its thread pairs stay matched.
            if (ok) ok = mbar_wait_warp(smem_u32(&s_full[j & 1]), (j >> 1) & 1, failed);
            const int key0 = (blk_lo + j) * KB + half * HC;
            const bool diagonal = key0 + HC - 1 > qpos;
            const uint32_t s_addr = lane_addr + (uint32_t)((j & 1) * KB + half * HC);
            // 16 scores at a time, read twice (for the maximum, for the exponentials): registers for two CTAs an SM
            auto scores = [&](int c0, uint32_t (&sr)[16]) {
                if (ok) {
                    tmem_ld_16(s_addr + (uint32_t)c0, sr);
                } else {
#pragma unroll
                    for (int c = 0; c < 16; ++c) sr[c] = 0u;
                }
                if (diagonal) {
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        if (key0 + c0 + c > qpos) sr[c] = 0xff800000u;     // -inf
                }
            };
            if (ok) tcgen05_fence_after();
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c0 = 0; c0 < HC; c0 += 16) {
                uint32_t sr[16];
                scores(c0, sr);
#pragma unroll
                for (int c = 0; c < 16; ++c) mx4[c & 3] = fmaxf(mx4[c & 3], __uint_as_float(sr[c]));
            }
            const float mx_own = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            xmax[((j & 1) * 2 + half) * QT + r] = mx_own;
            asm volatile("bar.sync %0, 64;" ::"r"(quarter + 1) : "memory");
            const float mx = fmaxf(mx_own, xmax[((j & 1) * 2 + (half ^ 1)) * QT + r]) * sl2;
            // (the reference maximum moves in large steps only: softmax does not depend on it, and results in tensor
            // memory are rarely rescaled)
            float m_new = m_run;
            if (m_run == -INFINITY || mx > m_run + RESCALE_STEP) m_new = mx;
            const bool rescale = m_run != -INFINITY && m_new != m_run;
            const float corr = rescale ? exp2_fast(m_run - m_new) : 1.0f;
            m_run = m_new;
            const float neg_m = m_new == -INFINITY ? 0.0f : -m_new;
            // the product of the block before has retired: P is free and the results may be touched
            if (ok && j >= 1) {
                ok = mbar_wait_warp(smem_u32(o_full), (j - 1) & 1, failed);
                if (ok) tcgen05_fence_after();
            }
            if (ok && __any_sync(0xffffffffu, rescale)) {
#pragma unroll
                for (int c0 = 0; c0 < 32 * ND; c0 += 16) {
                    uint32_t ob[16];
                    tmem_ld_16(lane_addr + O_COL + (uint32_t)(half * ND * 32 + c0), ob);
#pragma unroll
                    for (int i = 0; i < 16; ++i) ob[i] = __float_as_uint(__uint_as_float(ob[i]) * corr);
                    tmem_st_16(lane_addr + O_COL + (uint32_t)(half * ND * 32 + c0), ob);
                }
            }
            float rs0 = 0.0f, rs1 = 0.0f;
#pragma unroll
            for (int c0 = 0; c0 < HC; c0 += 16) {
                uint32_t sr[16], pk[8];
                scores(c0, sr);
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                    const float p0 = exp2_fast(fmaf(__uint_as_float(sr[c]), sl2, neg_m));
                    const float p1 = exp2_fast(fmaf(__uint_as_float(sr[c + 1]), sl2, neg_m));
                    rs0 += p0;
                    rs1 += p1;
                    pk[c >> 1] = pack2(p0, p1);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    st_shared_v4(smem_u32(p_s) + r * 128 + (((half * 4 + c0 / 8 + c) ^ (r & 7)) << 4), pk[4 * c], pk[4 * c + 1],
                                 pk[4 * c + 2], pk[4 * c + 3]);
            }
            l_run = l_run * corr + (rs0 + rs1);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(p_full));
        }
        // the row sum: both halves, in the words of a block behind the last: the other thread may not have read the last
        // block's maximum yet
        xmax[((n_blocks & 1) * 2 + half) * QT + r] = l_run;
        asm volatile("bar.sync %0, 64;" ::"r"(quarter + 1) : "memory");
        l_all = l_run + xmax[((n_blocks & 1) * 2 + (half ^ 1)) * QT + r];
        if (ok && n_blocks > 0) ok = mbar_wait_warp(smem_u32(o_full), (n_blocks - 1) & 1, failed);
        tcgen05_fence_after();
        if (!ok && lane == 0) prb_set_status(p.status, PRB_S_WAIT_TIMEOUT, 45, blockIdx.x, warp);
    } else {
        // ------------------------------------------------- codes to operands
        const int t = (warp - 2 - SOFTMAX) * 32 + lane;
        const int key8 = lane & 7, w = lane >> 3;                 // a key of 8, a word of a group's 4: no bank twice
        // One block's keys (KIND 0) or values: 8 keys x a group's 4 words at a time, 8 (keys) x NG of them, an eighth for each
        // warp; all words are asked for before the first is used.
        auto convert = [&](int j, auto kind_t) -> bool {
            constexpr int KIND = decltype(kind_t)::value;
            const int rs = j % RAW_STAGES, st = j % STAGES, key0 = (blk_lo + j) * KB;
            bool fine = KIND == 0 ? mbar_wait_warp(smem_u32(&raw_full[rs]), (j / RAW_STAGES) & 1, failed) : true;
            if (fine) fine = mbar_wait_warp(smem_u32(KIND == 0 ? &k_empty[st] : &v_empty[st]), ((j / STAGES) & 1) ^ 1, failed);
            if (!fine) {
                if (lane == 0) prb_set_status(p.status, PRB_S_WAIT_TIMEOUT, 46, blockIdx.x, j);
                return false;
            }
            const uint8_t* src = raw + rs * 2 * RAW + KIND * RAW;
            const uint32_t stage = smem_u32(ring + (size_t)st * STAGE) + KIND * 2 * ND * TILE;
            constexpr int TASKS = 8 * NG / DEQUANT;
            uint32_t word[TASKS], pair[TASKS];
#pragma unroll
            for (int i = 0; i < TASKS; ++i) {
                const int task = (t >> 5) + i * DEQUANT, g = task >> 3, key = (task & 7) * 8 + key8;
                word[i] = pair[i] = 0u;                                   // (channels beyond the head's are zero)
                if (g * 32 + w * 8 < head_dim) {
                    word[i] = *reinterpret_cast<const uint32_t*>(src + g * KB * 16 + key * (head_dim - g * 32 >= 32 ? 16 : 8) + w * 4);
                    pair[i] = *reinterpret_cast<const uint32_t*>(src + KB * (head_dim / 2) + (key * ng + g) * 4);
                }
            }
            // Keys that not all rows see, before the conversion (a branch within it keeps tasks from overlapping: 512 tokens at
            // 8,000 of 32 heads over 8 x 128 224 us instead of 188).
            if (KIND == 1 && key0 + KB - 1 > pos_lo) {
#pragma unroll
                for (int i = 0; i < TASKS; ++i) {
                    const int task = (t >> 5) + i * DEQUANT, g = task >> 3, key = (task & 7) * 8 + key8;
                    if (key0 + key <= pos_lo) continue;
                    // seen by none (stale), or by some, and then it may be no number: NaN or an infinity, or one from half a
                    // step past the largest of bfloat16 on
                    const float step = __uint_as_float(pair[i] << 16), middle = __uint_as_float(pair[i] & 0xffff0000u);
                    float most = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        most = fmaxf(most, fabsf(fmaf(step, (float)((int)((word[i] >> (4 * e)) & 15u) - 8), middle)));
                    const bool number = fabsf(step) < INFINITY && fabsf(middle) < INFINITY && most < 3.3961775e38f;
                    if (!number && key0 + key <= pos_hi) atomicMin(&poison[g], key0 + key);
                    if (!number || key0 + key > pos_hi) pair[i] = 0u;
                }
            }
            // (channels i and i + 4 of a word's 8 lie together, as one shift and one mask take them from it: the queries are
            // laid out alike, and the results' channels are put right when they are stored)
#pragma unroll
            for (int i = 0; i < TASKS; ++i) {
                const int task = (t >> 5) + i * DEQUANT, g = task >> 3, key = (task & 7) * 8 + key8;
                const int chunk = (g & 1) * 4 + w;                        // of the row's 8 pieces of 8 channels
                const uint32_t at = stage + (g >> 1) * TILE + key * 128 + ((chunk ^ (key & 7)) << 4);
                uint32_t hi[4];
                if (KIND == 1) {
                    // middle + step * (c - 8), rounded once
                    const uint32_t step = __byte_perm(pair[i], 0u, 0x1010), middle = __byte_perm(pair[i], 0u, 0x3232);
                    const __nv_bfloat162 off = __floats2bfloat162_rn(136.0f, 136.0f);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t u = ((word[i] >> (4 * e)) & 0x000f000fu) | p.magic;
                        const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&step),
                                                         __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), off),
                                                         *reinterpret_cast<const __nv_bfloat162*>(&middle));
                        hi[e] = *reinterpret_cast<const uint32_t*>(&v);
                    }
                    st_shared_v4(at, hi[0], hi[1], hi[2], hi[3]);
                } else {
                    const float step = __uint_as_float(pair[i] << 16);
                    const float base = fmaf(step, -136.0f, __uint_as_float(pair[i] & 0xffff0000u));   // (codes come as 128 + c)
                    uint32_t lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t u = ((word[i] >> (4 * e)) & 0x000f000fu) | p.magic;
                        const float x0 = fmaf(step, __uint_as_float(u << 16), base);
                        const float x1 = fmaf(step, __uint_as_float(u & 0xffff0000u), base);
                        hi[e] = pack2(x0, x1);
                        lo[e] = pack2(x0 - __uint_as_float(hi[e] << 16), x1 - __uint_as_float(hi[e] & 0xffff0000u));
                    }
                    st_shared_v4(at, hi[0], hi[1], hi[2], hi[3]);
                    st_shared_v4(at + ND * TILE, lo[0], lo[1], lo[2], lo[3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (KIND == 1) mbar_arrive(smem_u32(&raw_empty[rs]));
                mbar_arrive(smem_u32(KIND == 0 ? &k_full[st] : &v_full[st]));
            }
            return true;
        };
        // (a block's values after the next one's keys, which are wanted first)
        for (int j = 0; j <= n_blocks && ok; ++j) {
            if (j < n_blocks) ok = convert(j, std::integral_constant<int, 0>());
            if (ok && j > 0) ok = convert(j - 1, std::integral_constant<int, 1>());
        }
    }

    // --------------------------------------------------------------------- results
    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const bool all_fine = *failed == 0;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    constexpr int HD = D / 2;
    const int row = first + min(r, rows - 1), tk = row / p.hpg, qpos = pos0 + tk;
    __nv_bfloat16* dst = p.out + (long)(row0 + tk) * p.out_stride + (long)(hk * p.hpg + row - tk * p.hpg) * head_dim;
    // 8 channels from ch on, x in the operands' order (0, 4, 1, 5, 2, 6, 3, 7)
    auto store8 = [&](int ch, const float (&x)[8], float inv, bool bad) {
        const float nan = __int_as_float(0x7fc00000);
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = bad ? nan : x[2 * i] * inv;
            y[i + 4] = bad ? nan : x[2 * i + 1] * inv;
        }
        *reinterpret_cast<uint4*>(dst + ch) = make_uint4(pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7]));
    };
    if (p.parts == 1) {
        if (softmax && all_fine) {
            const float inv = l_all > 0.0f || l_all != l_all ? 1.0f / l_all : 0.0f;
#pragma unroll
            for (int c0 = 0; c0 < HD; c0 += 16) {
                uint32_t ob[16];
                tmem_ld_16(lane_addr + O_COL + (uint32_t)(half * HD + c0), ob);
                if (r < rows) {
#pragma unroll
                    for (int c = 0; c < 16; c += 8) {
                        const int ch = half * HD + c0 + c;
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(ob[c + i]);
                        if (ch < head_dim) store8(ch, x, inv, qpos >= poison[ch >> 5]);
                    }
                }
            }
        }
    } else {
        // parts: results [channel][row], maxima, sums and poison of each in its own shared memory; every CTA of the cluster
        // puts a share of the channels together, in the keys' order
        float* state = reinterpret_cast<float*>(ring);
        if (softmax) {
            if (n_blocks > 0 && all_fine) {
#pragma unroll
                for (int c0 = 0; c0 < HD; c0 += 16) {
                    uint32_t ob[16];
                    tmem_ld_16(lane_addr + O_COL + (uint32_t)(half * HD + c0), ob);
#pragma unroll
                    for (int i = 0; i < 16; ++i) state[(half * HD + c0 + i) * QT + r] = __uint_as_float(ob[i]);
                }
            }
            if (half == 0) {
                state_m[r] = all_fine && n_blocks > 0 ? m_run : -INFINITY;
                state_l[r] = all_fine && n_blocks > 0 ? l_all : 0.0f;
            }
        }
        cluster_sync_all();
        if (softmax) {
            float weight[MAX_PARTS], top = -INFINITY, sum = 0.0f;
            for (int z = 0; z < p.parts; ++z) top = fmaxf(top, lds_cluster(cluster_addr(smem_u32(state_m + r), z)));
#pragma unroll
            for (int z = 0; z < MAX_PARTS; ++z) {
                weight[z] = -1.0f;                                 // (no keys of the row's: there may be no results)
                if (z < p.parts) {
                    const float mz = lds_cluster(cluster_addr(smem_u32(state_m + r), z));
                    if (mz != -INFINITY) weight[z] = exp2_fast(mz - top);
                    sum += fmaxf(weight[z], 0.0f) * lds_cluster(cluster_addr(smem_u32(state_l + r), z));
                }
            }
            const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
            const int share = HD / p.parts;                        // (a multiple of 8: 32 or 64 channels, up to 4 parts)
            for (int c = 0; c < share; c += 8) {
                const int ch = half * HD + rank * share + c;
                float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int z = 0; z < MAX_PARTS; ++z)
                    if (z < p.parts && weight[z] >= 0.0f) {        // (0 times NaN goes on)
                        const uint32_t at = cluster_addr(smem_u32(state + (size_t)ch * QT + r), z);
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = fmaf(weight[z], lds_cluster(at + i * QT * 4), x[i]);
                    }
                // (the last part holds the keys that not all rows see, and with them the poison)
                bool bad = false;
                for (int z = 0; z < p.parts; ++z) {
                    int key;
                    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(key) : "r"(cluster_addr(smem_u32(poison + (ch >> 5)), z)) : "memory");
                    bad = bad || qpos >= key;
                }
                if (r < rows && all_fine && ch < head_dim) store8(ch, x, inv, bad);
            }
        }
        cluster_sync_all();                                        // nobody leaves while its results may be read
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

template <int ND, bool FULL> int launch_tile(const Params& p, cudaStream_t stream) {
    cudaError_t e = prb_allow_shared<attention_4bit_tile_kernel<ND, FULL>>((int)Sizes<ND>::SMEM);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long)p.n_tiles * p.kv_heads * p.subs * p.parts));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Sizes<ND>::SMEM;
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
    e = cudaLaunchKernelEx(&cfg, attention_4bit_tile_kernel<ND, FULL>, p);
    return e == cudaSuccess ? 0 : (int)e;
}
}  // namespace

// Whether the tensor-memory kernel takes a call (see prb_attention_4bit).
bool prb_attention_4bit_tile_takes(int head_dim, int page_size, int window, const void* q, long q_stride, const void* out,
                                   long out_stride) {
    return cache4::takes(head_dim, page_size) && window == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 &&
           q_stride % 8 == 0 && out_stride % 8 == 0;
}

int prb_attention_4bit_tile(void* out, long out_stride, const void* q, long q_stride, const uint8_t* k_tiles,
                            const uint8_t* v_tiles, const int* block_table, const int* positions, const int* tile_req,
                            const int* tile_row0, const int* tile_rows, const int* tile_count, int n_tiles, long rows,
                            int n_tokens, int n_requests, int kv_heads, int hpg, int head_dim, int page_size, int max_pages,
                            int num_pages, float scale, int max_context, int parts, int* status, cudaStream_t stream) {
    const long subs = (rows + QT - 1) / QT, units = (long)n_tiles * kv_heads * subs;
    if (units > 0x7fffffffL / MAX_PARTS) return PRB_E_SIZE;
    Params p{(__nv_bfloat16*)out, out_stride, (const __nv_bfloat16*)q, q_stride, k_tiles, v_tiles, block_table, positions,
             tile_req, tile_row0, tile_rows, tile_count, n_tokens, n_requests, n_tiles, (int)subs, 1, kv_heads, hpg, head_dim,
             page_size, max_pages, num_pages, cache4::tile_bytes(head_dim, page_size),
             page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : 16, scale, 0x43004300u, status};
    const int blocks = (max_context + KB - 1) / KB;
    // Parts of a tile's keys while all CTAs still run side by side (two an SM at head size 64, one at 128), each of at least
    // eight blocks: 128 tokens at 1,000 of 12 heads (12 units) 27.4 us in one part, 20.3 in two, 16.0 in four; 2 x 1,024
    // tokens of 12 heads (192 units) 36.1, 37.9 and 48.5; 512 tokens at 8,000 of 8 x 128 (128 units) 184, 196 and 219.
    // (Asked for by the call: 1, 2 or 4, whichever is not above it.)
    const long slots = (head_dim <= 64 ? 2L : 1L) * prb_sm_count();
    while (p.parts < MAX_PARTS && units * p.parts * 2 <= slots && blocks >= p.parts * 8) p.parts *= 2;
    if (parts > 0) p.parts = parts >= 4 ? 4 : parts >= 2 ? 2 : 1;
    if (p.piece == KB && head_dim == 64) return launch_tile<1, true>(p, stream);
    if (p.piece == KB && head_dim == 128) return launch_tile<2, true>(p, stream);
    return head_dim <= 64 ? launch_tile<1, false>(p, stream) : launch_tile<2, false>(p, stream);
}
