// Drafted tokens against the target's probabilities.
//
// A request brings n drafted tokens x_1 .. x_n and the target's logits of n + 1 rows: row i (from 0) says what comes
// behind the i-th of them.  With p_i = softmax(row i / temperature), q_i what the draft drew x_{i+1} from and given
// uniform numbers u_i, v_i in [0, 1):
//   x_{i+1} stays while  u_i * q_i(x) < p_i(x)  and all before it stayed;
//   the token behind the last that stays is drawn by v of its row: from max(p - q, 0), scaled to 1, where a token was
//   refused (from p, should nothing be left), from p behind the last drafted one: the lowest index at which the
//   running sum passes v times the whole.
// Without probabilities of the draft q is 1 at the drafted token.  Temperature 0 or less: a token stays while it is the
// largest logit (the lowest index among equals, a NaN before all numbers), and the largest logit follows.
//
// One launch; a cluster of eight CTAs takes a request, each an eighth of the vocabulary, and they meet through
// distributed shared memory.  First all rows' maximum and sum of exponentials in 32 bits (or their largest logit), one read
// of the logits from memory, which is what bounds it: 64 requests of 5 rows of 50,257 are 64 MB.  That decides who stays, but
// for a u q next to its p, where the row's sum is taken again in 64 bits.  Then the one row that is
// drawn from, in 64 bits: the border between two tokens moves by the error of a running sum over the whole vocabulary, and
// in 32 bits one draw in some hundred would fall on the other side.  The row comes from the L2, where the first pass left
// it; its exponentials (exp64: 20 operations of 64 bits) are taken once and kept in shared memory where they fit.
// 256 threads, so that four CTAs fit an SM and the clusters of 64 requests run side by side.
//
// 64 requests of 5 rows of 50,257: 41 us, of which a CTA spends 13 to 17 on the rows (64 MB are 10 us' worth), 5 on who stays
// and 15 on the drawn row, where it waits for the others three times; without a draw (temperature 0) 22 us.  One request
// of 5 rows 20 us, of which 10 on the drawn row.
#include "common.cuh"
#include "ranges.cuh"
#include "tcgen05.cuh"

namespace {
constexpr int PARTS = 8, THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_ROWS = 32;
constexpr int BATCH = 7;                  // 16-byte loads of a thread at a time: a row of up to 57,344 in one go
constexpr int AHEAD = 8;                  // numbers of a thread asked for together in the second part
constexpr int KEPT = 8192;                // most exponentials of a CTA's share that are kept (64 KB)

struct VerifyArgs {
    int* tokens;
    int* accepted;
    const float* logits;
    long logits_stride;
    const int* row_start;
    const int* drafted;
    const float* draft_probs;
    long probs_stride;
    const float* uniforms;
    const float* temperature;
    int n_requests, n_rows, vocab;
    int* status;
};

struct Shared {
    // a row's (maximum, its index, sum of exponentials) by warp, then of the CTA in place 0
    float top[MAX_ROWS][WARPS], sum[MAX_ROWS][WARPS];
    int index[MAX_ROWS][WARPS];
    double part[2][WARPS], total[2];          // two sums take turns, so that one can be read while the next is made
};

__device__ __forceinline__ uint32_t at_rank(const void* p, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(tc5::smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float peer_f(const float* p, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at_rank(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ int peer_i(const int* p, int rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at_rank(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ double peer_d(const double* p, int rank) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at_rank(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// 2^x by the hardware approximation (relative error about 2^-22)
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// (largest value, lowest index among equals; a NaN is larger than any number, as for the greedy sampler)
__device__ __forceinline__ void better(float& v, int& i, float w, int k) {
    const bool number = v == v;
    if (w != w ? number || k < i : number && (w > v || (w == v && k < i))) {
        v = w;
        i = k;
    }
}

// e^x for x <= 0: x = k ln 2 + r with |r| <= ln 2 / 2, and Taylor's series of e^r to r^13 (what it leaves out is below
// 2^-57); 0 below e^-700.
__device__ __forceinline__ double exp64(double x) {
    const double k = rint(x * 1.4426950408889634);
    double r = fma(k, -0.6931471805599453, x);
    r = fma(k, -2.3190468138462996e-17, r);                 // (what ln 2 loses in 64 bits)
    double y = 1.0 / 6227020800.0;
    y = fma(y, r, 1.0 / 479001600.0);
    y = fma(y, r, 1.0 / 39916800.0);
    y = fma(y, r, 1.0 / 3628800.0);
    y = fma(y, r, 1.0 / 362880.0);
    y = fma(y, r, 1.0 / 40320.0);
    y = fma(y, r, 1.0 / 5040.0);
    y = fma(y, r, 1.0 / 720.0);
    y = fma(y, r, 1.0 / 120.0);
    y = fma(y, r, 1.0 / 24.0);
    y = fma(y, r, 1.0 / 6.0);
    y = fma(y, r, 0.5);
    y = fma(y, r, 1.0);
    y = fma(y, r, 1.0);
    if (!(x > -700.0)) return 0.0;                          // (-inf, whose r is no number, too)
    return y * __hiloint2double((1023 + (int)k) << 20, 0);
}

// AHEAD_ROWS: the next row's logits are asked for before a row is worked on, for launches that leave the registers for it.
template <bool AHEAD_ROWS>
__global__ void __cluster_dims__(PARTS, 1, 1) __launch_bounds__(THREADS, AHEAD_ROWS ? 2 : 4) verify_kernel(const VerifyArgs p) {
    __shared__ Shared s;
    extern __shared__ double kept_e[];       // [each] exponentials of the row that is drawn from
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int req = blockIdx.x / PARTS, rank = blockIdx.x % PARTS;
    prb_grid_launch_dependents();
    prb_grid_wait();
    const int r0 = p.row_start[req], r1 = p.row_start[req + 1], rows = r1 - r0;
    if (r0 < 0 || rows < 1 || rows > MAX_ROWS || r1 > p.n_rows) {         // (the whole cluster leaves)
        if (threadIdx.x == 0 && rank == 0) {
            prb_set_status(p.status, PRB_S_ROW_RANGE, r0, r1, p.n_rows);
            p.accepted[req] = 0;
        }
        // (what an earlier step left in its rows is not an answer; a range that leaves the tensor names no rows)
        if (r0 >= 0 && r1 <= p.n_rows)
            for (int r = r0 + rank * THREADS + (int)threadIdx.x; r < r1; r += PARTS * THREADS) p.tokens[r] = -1;
        return;
    }
    const float t = p.temperature[req];
    const bool greedy = !(t > 0.0f);
    // (of temperatures whose scale is 0 or no number in 32 bits the products below are none either: it stops before that, and
    // the sums of such rows are looked at in 64 bits)
    const float scale = greedy ? 1.0f : fminf(fmaxf(1.4426950408889634f / t, 1e-37f), 1e37f);
    const bool extreme = !(t > 1e-30f && t < 1e30f);
    // this CTA's tokens, and each warp's run of them
    const int each = (p.vocab + PARTS - 1) / PARTS;
    const int lo = min(rank * each, p.vocab), hi = min(lo + each, p.vocab);

    // ---------------------------------------------------------- every row: maximum, sum
    // 16 bytes at a time from the first such border on; up to three logits before it and behind the last one alone
    auto head_of = [&](int r) -> int {
        const float* x = p.logits + (long)(r0 + r) * p.logits_stride + lo;
        return min((int)((16 - ((uintptr_t)x & 15)) & 15) / 4, hi - lo);
    };
    // a thread's part of a row, all asked for before the first is used; -inf weighs nothing
    auto batch = [&](int r, int i, float (&v)[4 * BATCH]) {
        const int head = head_of(r), vecs = (hi - lo - head) / 4;
        const float4* body = reinterpret_cast<const float4*>(p.logits + (long)(r0 + r) * p.logits_stride + lo + head);
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            float4 w = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (i + k * THREADS < vecs) w = body[i + k * THREADS];
            v[4 * k] = w.x; v[4 * k + 1] = w.y; v[4 * k + 2] = w.z; v[4 * k + 3] = w.w;
        }
    };
    auto edge = [&](int r, float& v) -> int {
        const int head = head_of(r), tail = lo + head + (hi - lo - head) / 4 * 4;
        const int at = threadIdx.x < 4 ? (threadIdx.x < head ? lo + threadIdx.x : hi)
                                       : threadIdx.x < 8 ? min(tail + (int)threadIdx.x - 4, hi) : hi;
        v = at < hi ? p.logits[(long)(r0 + r) * p.logits_stride + at] : -INFINITY;
        return at;
    };
    float v[4 * BATCH], lone;
    int lone_at = 0;
    if (AHEAD_ROWS) {
        batch(0, threadIdx.x, v);
        lone_at = edge(0, lone);
    }
    for (int r = 0; r < rows; ++r) {
        float top = -INFINITY, sum = 0.0f;
        int index = 0x7fffffff;
        auto sums = [&](const auto& v) {
            constexpr int n = sizeof(v) / sizeof(float);
            float now = top;
#pragma unroll
            for (int i = 0; i < n; ++i) now = fmaxf(now, v[i]);
            const float ref = now == -INFINITY ? 0.0f : now;
            sum *= exp2_fast((top - ref) * scale);
#pragma unroll
            for (int i = 0; i < n; ++i) sum += exp2_fast((v[i] - ref) * scale);
            top = now;
        };
        const int head = head_of(r), vecs = (hi - lo - head) / 4;
        auto take = [&](const float (&v)[4 * BATCH], int i) {
            if (!greedy) {
                sums(v);
                return;
            }
            // The largest first, then the lowest place that has it (places go up within a batch and from batch to batch): one
            // request of 4 rows of 50,257 takes 9.0 us a call, with `better` number by number 13.0.
            float quads[BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; ++k)
                quads[k] = max_nan(max_nan(v[4 * k], v[4 * k + 1]), max_nan(v[4 * k + 2], v[4 * k + 3]));
            float most = quads[0];
#pragma unroll
            for (int k = 1; k < BATCH; ++k) most = max_nan(most, quads[k]);
            const bool none = most != most;
            if (i >= vecs || !(none ? top == top : most > top || index == 0x7fffffff)) return;
            int at = 0;
            if (none) {
#pragma unroll
                for (int k = 4 * BATCH - 1; k >= 0; --k)
                    if (v[k] != v[k]) at = 4 * (k / 4) * THREADS + k % 4;
            } else {
#pragma unroll
                for (int k = 4 * BATCH - 1; k >= 0; --k)
                    if (v[k] == most) at = 4 * (k / 4) * THREADS + k % 4;
            }
            top = most;
            index = lo + head + 4 * i + at;
        };
        float next[4 * BATCH], next_lone = -INFINITY;
        int next_at = hi;
        if (!AHEAD_ROWS) {
            batch(r, threadIdx.x, v);
            lone_at = edge(r, lone);
        } else if (r + 1 < rows) {
            batch(r + 1, threadIdx.x, next);
            next_at = edge(r + 1, next_lone);
        }
        take(v, threadIdx.x);
        for (int i = threadIdx.x + BATCH * THREADS; i < vecs; i += BATCH * THREADS) {
            batch(r, i, v);
            take(v, i);
        }
        if (lone_at < hi) {
            const float one[1] = {lone};
            if (greedy) better(top, index, lone, lone_at);
            else sums(one);
        }
        if (AHEAD_ROWS) {
#pragma unroll
            for (int i = 0; i < 4 * BATCH; ++i) v[i] = next[i];
            lone = next_lone;
            lone_at = next_at;
        }
        // the warp's lanes
        const float own = top;
        if (greedy) {
            asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(own));
            index = (int)__reduce_min_sync(0xffffffffu, (unsigned)(own == top || own != own ? index : 0x7fffffff));
        } else {
            asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(own));
            const float ref = top == -INFINITY ? 0.0f : top;
            sum *= exp2_fast((own - ref) * scale);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (lane == 0) {
            s.top[r][warp] = top;
            s.sum[r][warp] = sum;
            s.index[r][warp] = index;
        }
    }
    __syncthreads();
    if (threadIdx.x < rows) {
        const int r = threadIdx.x;
        float top = s.top[r][0], sum = s.sum[r][0];
        int index = s.index[r][0];
        for (int w = 1; w < WARPS; ++w) {
            const float was = top, v = s.top[r][w];
            better(top, index, v, s.index[r][w]);
            if (!greedy) {
                const float ref = top == -INFINITY ? 0.0f : top;
                sum = sum * exp2_fast((was - ref) * scale) + s.sum[r][w] * exp2_fast((v - ref) * scale);
            }
        }
        s.top[r][0] = top;
        s.sum[r][0] = sum;
        s.index[r][0] = index;
    }
    cluster_sync_all();

    // the CTA's sum, then all CTAs'
    int turn = 1;
    auto meet = [&](double v) -> double {
        turn ^= 1;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) s.part[turn][warp] = v;
        __syncthreads();
        if (threadIdx.x == 0) {
            double a = 0.0;
            for (int w = 0; w < WARPS; ++w) a += s.part[turn][w];
            s.total[turn] = a;
        }
        cluster_sync_all();
        double all = 0.0;
        for (int c = 0; c < PARTS; ++c) all += peer_d(&s.total[turn], c);
        return all;
    };
    // -------------------------------- who stays: lane i looks at row i, every warp by itself
    float top = -INFINITY;
    int best = 0x7fffffff;
    bool stays = false, unsure = false;
    const double inverse = greedy ? 0.0 : 1.0 / (double)t;
    // What the sum in 32 bits may be off by, of itself.  An exponent is off by 2^-23 of itself (the scale's rounding, the
    // product's), and a term of exponent -x weighs 2^-x, so a whole row of them by less than 32 x 2^-23; the exponential by
    // 2^-22, a sum of n terms one after the other by n 2^-24.  Twice that and more is called next to the border.
    const double doubt = (64 + each / THREADS) * 2.384185791015625e-07;
    if (lane < rows) {
        float part[PARTS], sum = 0.0f;
#pragma unroll
        for (int z = 0; z < PARTS; ++z) {
            part[z] = peer_f(&s.top[lane][0], z);
            better(top, best, part[z], peer_i(&s.index[lane][0], z));
        }
        const float ref = top == -INFINITY ? 0.0f : top;
        if (!greedy) {
#pragma unroll
            for (int z = 0; z < PARTS; ++z) sum += peer_f(&s.sum[lane][0], z) * exp2_fast((part[z] - ref) * scale);
            if (!(fabsf(top) < INFINITY && sum > 0.0f && sum < INFINITY) && rank == 0 && warp == 0)
                prb_set_status(p.status, PRB_S_LOGITS, r0 + lane, req, 0);
        } else if (!(fabsf(top) < INFINITY) && rank == 0 && warp == 0) {
            prb_set_status(p.status, PRB_S_LOGITS, r0 + lane, req, 0);
        }
        if (lane + 1 < rows) {
            const int x = p.drafted[r0 + lane];
            if (x < 0 || x >= p.vocab) {
                if (rank == 0 && warp == 0) prb_set_status(p.status, PRB_S_TOKEN_RANGE, r0 + lane, x, p.vocab);
            } else if (greedy) {
                stays = x == best;
            } else {
                const double mine = exp64(((double)p.logits[(long)(r0 + lane) * p.logits_stride + x] - (double)ref) * inverse);
                const double theirs = p.draft_probs ? (double)p.draft_probs[(long)(r0 + lane) * p.probs_stride + x] : 1.0;
                const double bar = (double)p.uniforms[2 * (r0 + lane)] * theirs * (double)sum;
                stays = bar < mine;
                unsure = extreme || fabs(bar - mine) < doubt * mine;
            }
        }
    }
    int kept = __ffs(~__ballot_sync(0xffffffffu, stays)) - 1;             // (row rows - 1 never stays)
    // Next to the border the row's sum is taken again, in 64 bits (one row in some ten thousand; all CTAs come to the same
    // answers, since they added the same numbers in the same order).
    unsigned open = __ballot_sync(0xffffffffu, unsure);
    while (open != 0 && __ffs(open) - 1 <= kept) {
        const int r = __ffs(open) - 1;
        open &= open - 1;
        const float* x = p.logits + (long)(r0 + r) * p.logits_stride;
        const double ref = (double)__shfl_sync(0xffffffffu, top, r);
        double v = 0.0;
        for (int i = lo + threadIdx.x; i < hi; i += THREADS) v += exp64(((double)x[i] - ref) * inverse);
        const double whole = meet(v);
        if (lane == r) {
            const int token = p.drafted[r0 + r];
            const double theirs = p.draft_probs ? (double)p.draft_probs[(long)(r0 + r) * p.probs_stride + token] : 1.0;
            stays = (double)p.uniforms[2 * (r0 + r)] * theirs * whole < exp64(((double)x[token] - ref) * inverse);
        }
        kept = __ffs(~__ballot_sync(0xffffffffu, stays)) - 1;
    }
    const int row = r0 + kept;
    const bool refused = kept + 1 < rows;
    int chosen = __shfl_sync(0xffffffffu, best, kept);
    top = __shfl_sync(0xffffffffu, top, kept);
    if (chosen >= p.vocab) chosen = 0;

    if (!greedy && fabsf(top) < INFINITY) {
        // ------------------------------------------------- the row that is drawn from, in 64 bits
        const float* x = p.logits + (long)row * p.logits_stride;
        const float* q = refused && p.draft_probs ? p.draft_probs + (long)row * p.probs_stride : nullptr;
        const int gone = refused && !p.draft_probs ? p.drafted[row] : -1;
        const int run = (hi - lo + WARPS - 1) / WARPS;
        const int w0 = min(lo + warp * run, hi), w1 = min(w0 + run, hi);
        const bool keep = each <= KEPT;
        if (q != nullptr)                                                 // (wanted once the sum below is known)
            for (int i = lo + 32 * threadIdx.x; i < hi; i += 32 * THREADS)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(q + i));
        auto raw = [&](int i) -> double { return exp64(((double)x[i] - (double)top) * inverse); };
        double v = 0.0;
        float ahead[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) ahead[k] = w0 + lane + 32 * k < w1 ? x[w0 + lane + 32 * k] : -INFINITY;
        for (int i0 = w0 + lane; i0 < w1; i0 += 32 * AHEAD) {
            float l[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                l[k] = ahead[k];
                ahead[k] = i0 + 32 * (k + AHEAD) < w1 ? x[i0 + 32 * (k + AHEAD)] : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const double e = exp64(((double)l[k] - (double)top) * inverse);
                if (keep && i0 + 32 * k < w1) kept_e[i0 + 32 * k - lo] = e;
                v += e;
            }
        }
        double whole = meet(v);
        // Behind a refused token: what the target's probability leaves over the draft's, in the kept ones' place.  Without one
        // the exponentials are the weights as they are.
        const double z = 1.0 / whole;
        bool less = refused;
        auto weight = [&](int i) -> double {
            if (keep) return kept_e[i - lo];
            const double e = raw(i);
            if (!less) return e;
            if (q != nullptr) return fmax(e * z - (double)q[i], 0.0);
            return i == gone ? 0.0 : e;
        };
        if (less) {
            v = 0.0;
            for (int i0 = w0 + lane; i0 < w1; i0 += 32 * AHEAD) {
                float said[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) said[k] = q != nullptr && keep && i0 + 32 * k < w1 ? q[i0 + 32 * k] : 0.0f;
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const int i = i0 + 32 * k;
                    if (i >= w1) break;
                    if (keep) {
                        const double e = kept_e[i - lo], w = q != nullptr ? fmax(e * z - (double)said[k], 0.0) : i == gone ? 0.0 : e;
                        kept_e[i - lo] = w;
                        v += w;
                    } else {
                        v += weight(i);
                    }
                }
            }
            whole = meet(v);
            if (!(whole > 0.0)) {                                         // nothing left: the target's own
                less = false;
                v = 0.0;
                for (int i = w0 + lane; i < w1; i += 32) {
                    const double e = raw(i);
                    if (keep) kept_e[i - lo] = e;
                    v += e;
                }
                whole = meet(v);
            }
        }
        const double want = (double)p.uniforms[2 * row + 1] * whole;
        // the CTA whose sums pass it, else the last that has any weight
        double before = 0.0;
        int owner = -1, final_owner = 0;
        double owner_before = 0.0;
        for (int c = 0; c < PARTS; ++c) {
            const double v = peer_d(&s.total[turn], c);
            if (v > 0.0) final_owner = c;
            if (owner < 0 && before + v > want) {
                owner = c;
                owner_before = before;
            }
            before += v;
        }
        const bool passes = owner >= 0;
        if (!passes) owner = final_owner;
        if (owner == rank) {
            double b = owner_before;
            int mine = -1, final_mine = 0;
            double mine_before = 0.0;
            for (int w = 0; w < WARPS; ++w) {
                const double v = s.part[turn][w];
                if (v > 0.0) final_mine = w;
                if (mine < 0 && passes && b + v > want) {
                    mine = w;
                    mine_before = b;
                }
                b += v;
            }
            const bool inside = mine >= 0;
            if (!inside) mine = final_mine;
            if (mine == warp) {
                // each lane a run of neighbours (of an odd length: no bank of shared memory twice at a time), then the lane
                // whose sums pass it goes through its own
                const int each_lane = ((w1 - w0 + 31) / 32) | 1;
                const int a = min(w0 + lane * each_lane, w1), b1 = min(a + each_lane, w1);
                double own = 0.0;
                int final_token = -1;
                for (int i = a; i < b1; ++i) {
                    const double w = weight(i);
                    own += w;
                    if (w > 0.0) final_token = i;
                }
                double up = own;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double below = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += below;
                }
                const unsigned over = __ballot_sync(0xffffffffu, inside && final_token >= 0 && mine_before + up > want);
                const unsigned any = __ballot_sync(0xffffffffu, final_token >= 0);
                // (rounding may leave nobody that passes it: then the last token with any weight)
                const int chosen_lane = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : 0;
                if (lane == chosen_lane) {
                    int found = final_token < 0 ? 0 : final_token;
                    double sum = mine_before + (up - own);
                    for (int i = a; over && i < b1; ++i) {
                        const double w = weight(i);
                        sum += w;
                        if (w > 0.0 && sum > want) {
                            found = i;
                            break;
                        }
                    }
                    p.tokens[row] = found;
                }
            }
        }
    } else if (rank == 0 && threadIdx.x == 0) {
        p.tokens[row] = chosen;
    }
    if (rank == 0) {
        for (int r = threadIdx.x; r < rows; r += THREADS)
            if (r != kept) p.tokens[r0 + r] = r < kept ? p.drafted[r0 + r] : -1;
        if (threadIdx.x == 0) p.accepted[req] = kept;
    }
    cluster_sync_all();                                                   // nobody leaves while its sums may be read
}
}  // namespace

PRB_API int prb_verify_drafts(int* tokens, int* accepted, const float* logits, long logits_stride, const int* row_start,
                              const int* drafted, const float* draft_probs, long probs_stride, const float* uniforms,
                              const float* temperature, int n_requests, int n_rows, int vocab, int* status,
                              cudaStream_t stream) {
    if (n_requests <= 0) return 0;                            // (requests of no rows are recorded by the kernel)
    if (n_rows < 0 || vocab <= 0 || n_requests > 0x7fffffff / PARTS) return PRB_E_SIZE;
    const long word = 4, width = vocab * word;
    if (!prb_apart({{tokens, n_rows * word}, {accepted, n_requests * word}, {status, 4 * word}},
                   {{row_start, (n_requests + 1) * word}, {drafted, n_rows * word}, {uniforms, 2 * n_rows * word},
                    {temperature, n_requests * word}, {logits, prb_span(n_rows, logits_stride * word, width)},
                    {draft_probs, prb_span(n_rows, probs_stride * word, width)}}))
        return PRB_E_OVERLAP;
    const VerifyArgs a{tokens, accepted, logits, logits_stride, row_start, drafted, draft_probs, probs_stride, uniforms,
                       temperature, n_requests, n_rows, vocab, status};
    const int each = (vocab + PARTS - 1) / PARTS;
    const size_t shared = each <= KEPT ? each * sizeof(double) : 0;
    // The next row asked for ahead takes some 110 registers instead of 60, so it is for launches of two CTAs an SM at most.
    // us without and with it, 5 rows of 50,257 logits at temperature 0.8: 32 requests 33.2 and 27.4, one request 19.9 either
    // way; but 64, where four CTAs an SM do more, 41.3 and 52.0.
    const bool ahead = (long)n_requests * PARTS <= 2L * prb_sm_count();
    cudaError_t e = ahead ? prb_allow_shared<verify_kernel<true>>(KEPT * (int)sizeof(double))
                          : prb_allow_shared<verify_kernel<false>>(KEPT * (int)sizeof(double));
    if (e != cudaSuccess) return (int)e;
    const dim3 grid((unsigned)n_requests * PARTS);
    e = ahead ? prb_launch_dependent(verify_kernel<true>, grid, dim3(THREADS), shared, stream, a)
              : prb_launch_dependent(verify_kernel<false>, grid, dim3(THREADS), shared, stream, a);
    return e == cudaSuccess ? 0 : (int)e;
}
