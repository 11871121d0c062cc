// Causal attention of prompt portions over a cache held in 4 bits (cache4.cuh) on the 5th-generation tensor cores.
// bfloat16, head sizes 64 and 128, pages of a multiple of 64 positions, no window.
//
// One CTA takes up to 128 rows (tokens times the query heads of one key/value head) of a tile and walks the keys in
// blocks of 64, or one of the parts of them (parts are a cluster and meet through distributed shared memory).  Warps:
//   0      producer: bulk copies of a block's codes, steps and middles (5 KB at head size 64 for keys and values, where
//          bfloat16 is 16) into a ring of raw stages;
//   1      allocates tensor memory; one thread issues tcgen05.mma: S = Q K^T (128 x 64), O += P V;
//   2-9    softmax: two threads a row, each 32 of a block's 64 scores and half of the output's channels;
//   10-13  turn codes into operands in the swizzled layout, once for all 128 rows.
// Values become bfloat16 (2^-8 of a value, as a bfloat16 cache would hold it, on top of the cache's own rounding).  Keys
// become the sum of two bfloat16 numbers and take two products: a key's rounding moves a score by the product of the
// query's and the key's lengths times it, which at ordinary scores is several times what P's rounding costs, and the tensor
// cores wait for the softmax anyway.
//
// What lies behind the tile's last position (stale pages, NaN) becomes zeros.  A key that the tile's later tokens see and
// its earlier ones do not may read back as NaN: it becomes zeros too, and the rows that see it are made NaN in the channels
// of its group at the end, since a product would spread it over all rows.
//
// Every wait is bounded: where one gives up the status word says so, nothing more is stored, copies in flight are waited
// for, tensor memory is freed.
#include "cache4.cuh"
#include "tcgen05.cuh"

namespace {
using namespace tc5;

constexpr int QT = 128, KB = 64;
constexpr int SOFTMAX = 8, DEQUANT = 4, WARPS = 2 + SOFTMAX + DEQUANT, THREADS = WARPS * 32;
constexpr int RAW_STAGES = 2, STAGES = 2, MAX_PARTS = 4;
constexpr int P_BYTES = QT * KB * 2;
constexpr float RESCALE_STEP = 8.0f;         // a row's reference maximum moves only by more than this (log2 units)

// ND: head size / 64.
template <int ND> struct Sizes {
    static constexpr int D = 64 * ND, NG = 2 * ND;
    static constexpr int RAW = KB * (D / 2 + 4 * NG);           // bytes of a block's keys (and of its values)
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
    int kv_heads, hpg, page_size, max_pages, num_pages, tile_bytes;
    float scale;
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
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
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

template <int ND>
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
    uint64_t* kv_full = raw_empty + RAW_STAGES;  // [STAGES] dequant -> MMA
    uint64_t* kv_empty = kv_full + STAGES;       // MMA -> dequant
    uint64_t* s_full = kv_empty + STAGES;        // [2] scores ready
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

    if (threadIdx.x == 0) {
        for (int s = 0; s < RAW_STAGES; ++s) {
            mbar_init(smem_u32(&raw_full[s]), 1);
            mbar_init(smem_u32(&raw_empty[s]), DEQUANT);
        }
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&kv_full[s]), DEQUANT);
            mbar_init(smem_u32(&kv_empty[s]), 1);
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
        int j = 0;
        int page = n_blocks > 0 ? table[blk_lo * KB / p.page_size] : 0;
        for (; j < n_blocks; ++j) {
            const int st = j % RAW_STAGES, key0 = (blk_lo + j) * KB;
            ok = mbar_wait_warp(smem_u32(&raw_empty[st]), ((j / RAW_STAGES) & 1) ^ 1, failed);
            if (!ok) {
                if (lane == 0) prb_set_status(p.status, PRB_S_WAIT_TIMEOUT, 43, blockIdx.x, j);
                break;
            }
            const uint32_t fb = smem_u32(&raw_full[st]);
            const bool fine = page >= 0 && page < p.num_pages;
            const int at = key0 % p.page_size;
            if (lane == 0) {
                // (a page that is none: recorded, the stage keeps what it held, and the tile's result is not to be used)
                if (!fine) prb_set_status(p.status, PRB_S_PAGE_RANGE, row0, key0, page);
                mbar_expect_tx(fb, fine ? 2 * RAW : 0);
            }
            __syncwarp();
            const size_t from = fine ? ((size_t)page * p.kv_heads + hk) * (size_t)p.tile_bytes : 0;
            const uint32_t dst = smem_u32(raw) + st * 2 * RAW;
            if (fine && p.page_size == KB) {
                if (lane < 2) bulk_load(dst + lane * RAW, (lane ? p.v_tiles : p.k_tiles) + from, RAW, fb);
            } else if (fine && lane < 2 * (NG + 1)) {
                // lane i: copy i / 2 (a group's codes, or the pairs) of keys or values
                const int c = lane >> 1;
                const uint8_t* src = (lane & 1 ? p.v_tiles : p.k_tiles) + from;
                const uint32_t to = dst + (lane & 1) * RAW + c * KB * 16;
                if (c < NG)
                    bulk_load(to, src + c * p.page_size * 16 + at * 16, KB * 16, fb);
                else
                    bulk_load(to, src + p.page_size * (D / 2) + at * NG * 4, KB * NG * 4, fb);
            }
            __syncwarp();
            if (j + 1 < n_blocks) page = table[(key0 + KB) / p.page_size];
        }
        if (!ok) {
            for (int jj = j > RAW_STAGES ? j - RAW_STAGES : 0; jj < j; ++jj)      // copies still on their way
                for (uint32_t i = 0; i < WAIT_LIMIT; ++i)
                    if (mbar_try_wait(smem_u32(&raw_full[jj % RAW_STAGES]), (jj / RAW_STAGES) & 1)) break;
            __syncwarp();
        }
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
            }
            __syncwarp();
        };
        if (n_blocks > 0) {
            ok = mbar_wait_warp(smem_u32(q_full), 0, failed);
            if (ok) ok = mbar_wait_warp(smem_u32(&kv_full[0]), 0, failed);
            if (ok) {
                tcgen05_fence_after();
                issue_scores(0);
            }
            for (int j = 0; j < n_blocks && ok; ++j) {
                if (j + 1 < n_blocks) {
                    ok = mbar_wait_warp(smem_u32(&kv_full[(j + 1) % STAGES]), ((j + 1) / STAGES) & 1, failed);
                    if (!ok) break;
                    tcgen05_fence_after();
                    issue_scores(j + 1);
                }
                ok = mbar_wait_warp(smem_u32(p_full), j & 1, failed);
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
                    umma_commit(smem_u32(&kv_empty[j % STAGES]));
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
            const __nv_bfloat16* src = p.q + (long)(row0 + tk) * p.q_stride + (long)(hk * p.hpg + row - tk * p.hpg) * D;
#pragma unroll
            for (int c = 0; c < 4 * ND; ++c) {
                const int ci = half * 4 * ND + c;
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (row_ok) w = *reinterpret_cast<const uint4*>(src + ci * 8);
                st_shared_v4(smem_u32(q_s) + (ci >> 3) * QT * 128 + r * 128 + (((ci & 7) ^ (r & 7)) << 4), w.x, w.y, w.z, w.w);
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
            uint32_t sr[HC];
            if (ok) {
                tcgen05_fence_after();
                tmem_ld_32x32(lane_addr + (uint32_t)((j & 1) * KB + half * HC), sr);
            } else {
#pragma unroll
                for (int c = 0; c < HC; ++c) sr[c] = 0u;
            }
            const int key0 = (blk_lo + j) * KB + half * HC;
            if (key0 + HC - 1 > qpos) {
#pragma unroll
                for (int c = 0; c < HC; ++c)
                    if (key0 + c > qpos) sr[c] = 0xff800000u;              // -inf
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < HC; c += 4)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx4[e] = fmaxf(mx4[e], __uint_as_float(sr[c + e]));
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
            uint32_t pk[HC / 2];
            float rs0 = 0.0f, rs1 = 0.0f;
#pragma unroll
            for (int c = 0; c < HC; c += 2) {
                const float p0 = exp2_fast(fmaf(__uint_as_float(sr[c]), sl2, neg_m));
                const float p1 = exp2_fast(fmaf(__uint_as_float(sr[c + 1]), sl2, neg_m));
                rs0 += p0;
                rs1 += p1;
                pk[c >> 1] = pack2(p0, p1);
            }
            l_run = l_run * corr + (rs0 + rs1);
            // the product of the block before has retired: P is free and the results may be touched
            if (ok && j >= 1) {
                ok = mbar_wait_warp(smem_u32(o_full), (j - 1) & 1, failed);
                if (ok) tcgen05_fence_after();
            }
            if (ok && __any_sync(0xffffffffu, rescale)) {
#pragma unroll
                for (int a = 0; a < ND; ++a) {
                    uint32_t ob[32];
                    tmem_ld_32x32(lane_addr + O_COL + (uint32_t)((half * ND + a) * 32), ob);
#pragma unroll
                    for (int i = 0; i < 32; ++i) ob[i] = __float_as_uint(__uint_as_float(ob[i]) * corr);
                    tmem_st_32x32(lane_addr + O_COL + (uint32_t)((half * ND + a) * 32), ob);
                }
            }
#pragma unroll
            for (int c = 0; c < HC / 8; ++c)
                st_shared_v4(smem_u32(p_s) + r * 128 + (((half * 4 + c) ^ (r & 7)) << 4), pk[4 * c], pk[4 * c + 1],
                             pk[4 * c + 2], pk[4 * c + 3]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(p_full));
        }
        // the row sum: both halves
        xmax[half * QT + r] = l_run;
        asm volatile("bar.sync %0, 64;" ::"r"(quarter + 1) : "memory");
        l_all = half == 0 ? l_run + xmax[QT + r] : xmax[r] + l_run;
        if (ok && n_blocks > 0) ok = mbar_wait_warp(smem_u32(o_full), (n_blocks - 1) & 1, failed);
        tcgen05_fence_after();
        if (!ok && lane == 0) prb_set_status(p.status, PRB_S_WAIT_TIMEOUT, 45, blockIdx.x, warp);
    } else {
        // ------------------------------------------------- codes to operands
        const int t = (warp - 2 - SOFTMAX) * 32 + lane;
        const int key8 = lane & 7, w = lane >> 3;                 // a key of 8, a word of a group's 4: no bank twice
        for (int j = 0; j < n_blocks; ++j) {
            const int rs = j % RAW_STAGES, st = j % STAGES, key0 = (blk_lo + j) * KB;
            ok = mbar_wait_warp(smem_u32(&raw_full[rs]), (j / RAW_STAGES) & 1, failed);
            if (ok) ok = mbar_wait_warp(smem_u32(&kv_empty[st]), ((j / STAGES) & 1) ^ 1, failed);
            if (!ok) {
                if (lane == 0) prb_set_status(p.status, PRB_S_WAIT_TIMEOUT, 46, blockIdx.x, j);
                break;
            }
            const uint8_t* src = raw + rs * 2 * RAW;
            const uint32_t stage = smem_u32(ring + (size_t)st * STAGE);
            // 8 keys x a group's 4 words at a time: 8 (keys) x NG of them, a quarter for each warp
#pragma unroll
            for (int kind = 0; kind < 2; ++kind)
#pragma unroll
                for (int i = 0; i < 2 * NG; ++i) {
                    const int task = (t >> 5) + i * DEQUANT, g = task >> 3, key = (task & 7) * 8 + key8;
                    const uint32_t word = *reinterpret_cast<const uint32_t*>(src + kind * RAW + g * KB * 16 + key * 16 + w * 4);
                    const uint32_t pair =
                        *reinterpret_cast<const uint32_t*>(src + kind * RAW + KB * (D / 2) + (key * NG + g) * 4);
                    float step = __uint_as_float(pair << 16), middle = __uint_as_float(pair & 0xffff0000u);
                    if (kind == 1 && key0 + key > pos_lo) {
                        // not seen by all rows: by none (stale), or by some, and then it may be no number
                        const bool number = fabsf(step) < INFINITY && fabsf(middle) < INFINITY;
                        if (!number && key0 + key <= pos_hi && w == 0) atomicMin(&poison[g], key0 + key);
                        if (!number || key0 + key > pos_hi) step = middle = 0.0f;
                    }
                    const float base = fmaf(step, -136.0f, middle);           // (the codes come as 128 + c)
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t u = ((word >> (4 * e)) & 0x000f000fu) | 0x43004300u;
                        x[e] = fmaf(step, __uint_as_float(u << 16), base);
                        x[e + 4] = fmaf(step, __uint_as_float(u & 0xffff0000u), base);
                    }
                    uint32_t hi[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) hi[e] = pack2(x[2 * e], x[2 * e + 1]);
                    const int chunk = (g & 1) * 4 + w;                        // of the row's 8 pieces of 8 channels
                    const uint32_t at = (g >> 1) * TILE + key * 128 + ((chunk ^ (key & 7)) << 4);
                    st_shared_v4(stage + (kind ? 2 * ND * TILE : 0) + at, hi[0], hi[1], hi[2], hi[3]);
                    if (kind == 0) {
                        uint32_t lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            lo[e] = pack2(x[2 * e] - __uint_as_float(hi[e] << 16),
                                          x[2 * e + 1] - __uint_as_float(hi[e] & 0xffff0000u));
                        st_shared_v4(stage + ND * TILE + at, lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&raw_empty[rs]));
                mbar_arrive(smem_u32(&kv_full[st]));
            }
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
    __nv_bfloat16* dst = p.out + (long)(row0 + tk) * p.out_stride + (long)(hk * p.hpg + row - tk * p.hpg) * D;
    auto store8 = [&](int ch, const float (&x)[8], float inv) {
        float y[8];
        const bool bad = qpos >= poison[ch >> 5];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = bad ? __int_as_float(0x7fc00000) : x[i] * inv;
        *reinterpret_cast<uint4*>(dst + ch) = make_uint4(pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7]));
    };
    if (p.parts == 1) {
        if (softmax && all_fine) {
            const float inv = l_all > 0.0f || l_all != l_all ? 1.0f / l_all : 0.0f;
#pragma unroll
            for (int a = 0; a < ND; ++a) {
                uint32_t ob[32];
                tmem_ld_32x32(lane_addr + O_COL + (uint32_t)((half * ND + a) * 32), ob);
                if (r < rows) {
#pragma unroll
                    for (int c = 0; c < 32; c += 8) {
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(ob[c + i]);
                        store8((half * ND + a) * 32 + c, x, inv);
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
                for (int a = 0; a < ND; ++a) {
                    uint32_t ob[32];
                    tmem_ld_32x32(lane_addr + O_COL + (uint32_t)((half * ND + a) * 32), ob);
#pragma unroll
                    for (int i = 0; i < 32; ++i) state[((half * ND + a) * 32 + i) * QT + r] = __uint_as_float(ob[i]);
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
                weight[z] = 0.0f;
                if (z < p.parts) {
                    const float mz = lds_cluster(cluster_addr(smem_u32(state_m + r), z));
                    weight[z] = mz == -INFINITY ? 0.0f : exp2_fast(mz - top);
                    sum += weight[z] * lds_cluster(cluster_addr(smem_u32(state_l + r), z));
                }
            }
            const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
            const int share = HD / p.parts;                        // (a multiple of 8: 32 or 64 channels, up to 4 parts)
            for (int c = 0; c < share; c += 8) {
                const int ch = half * HD + rank * share + c;
                float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int z = 0; z < MAX_PARTS; ++z)
                    if (z < p.parts && weight[z] > 0.0f) {
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
                if (r < rows && all_fine) {
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = bad ? __int_as_float(0x7fc00000) : x[i] * inv;
                    *reinterpret_cast<uint4*>(dst + ch) =
                        make_uint4(pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7]));
                }
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

template <int ND> int launch_tile(const Params& p, cudaStream_t stream) {
    cudaError_t e = prb_allow_shared<attention_4bit_tile_kernel<ND>>((int)Sizes<ND>::SMEM);
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
    e = cudaLaunchKernelEx(&cfg, attention_4bit_tile_kernel<ND>, p);
    return e == cudaSuccess ? 0 : (int)e;
}
}  // namespace

// Whether the tensor-memory kernel takes a call (see prb_attention_4bit).
bool prb_attention_4bit_tile_takes(int head_dim, int page_size, int window, const void* q, long q_stride, const void* out,
                                   long out_stride) {
    return (head_dim == 64 || head_dim == 128) && page_size % KB == 0 && window == 0 && (uintptr_t)q % 16 == 0 &&
           (uintptr_t)out % 16 == 0 && q_stride % 8 == 0 && out_stride % 8 == 0;
}

int prb_attention_4bit_tile(void* out, long out_stride, const void* q, long q_stride, const uint8_t* k_tiles,
                            const uint8_t* v_tiles, const int* block_table, const int* positions, const int* tile_req,
                            const int* tile_row0, const int* tile_rows, const int* tile_count, int n_tiles, long rows,
                            int n_tokens, int n_requests, int kv_heads, int hpg, int head_dim, int page_size, int max_pages,
                            int num_pages, float scale, int max_context, int parts, int* status, cudaStream_t stream) {
    const long subs = (rows + QT - 1) / QT, units = (long)n_tiles * kv_heads * subs;
    if (units > 0x7fffffffL / MAX_PARTS) return PRB_E_SIZE;
    Params p{(__nv_bfloat16*)out, out_stride, (const __nv_bfloat16*)q, q_stride, k_tiles, v_tiles, block_table, positions,
             tile_req, tile_row0, tile_rows, tile_count, n_tokens, n_requests, n_tiles, (int)subs, 1, kv_heads, hpg, page_size,
             max_pages, num_pages, cache4::tile_bytes(head_dim, page_size), scale, status};
    const int blocks = (max_context + KB - 1) / KB;
    while (p.parts < MAX_PARTS && units * p.parts < 4L * prb_sm_count() && blocks >= p.parts * 8) p.parts *= 2;
    if (parts > 0) p.parts = parts >= 4 ? 4 : parts >= 2 ? 2 : 1;
    return head_dim == 64 ? launch_tile<1>(p, stream) : launch_tile<2>(p, stream);
}
