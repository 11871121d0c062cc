// Rows of keys and values into a cache held in 4 bits, and back (cache4.cuh has the layout).
//
// A decode step's 64 tokens of 12 heads of 64 are bound by the launch (2.5 us in, 2.0 us back).  2,048 tokens of 25 heads
// go in at 12.7 us, bound by the instructions of the rounding (17 MB move, 2.6 us' worth), and back at 8.6 us (30 MB, 4.6 us'
// worth).  Four threads share a group of 32 channels, 8 channels (16 bytes of
// bfloat16, one 32-bit word of codes) each; neighbouring threads take neighbouring groups of one token, so a
// warp reads 512 bytes in a row.  The smallest and the largest number of a group meet in two shuffles.
//
// Codes are those of exact arithmetic.  (x - middle) / step is taken in 32 bits, which is off by less than
// 2e-6; a quotient next to the border of two codes (borders are common: bfloat16 numbers are short) is decided
// by the sign of (x - middle) - border * step, which one fused multiply-add gives exactly, with what the
// difference's own rounding left out behind it.  Step and middle are taken in 64 bits, two operations a group.
// A group that holds an infinity or a NaN reads back as NaN.
#include "cache4.cuh"
#include "ranges.cuh"

namespace {
using cache4::GROUP;

struct RowArgs {
    uint8_t* tiles[2];              // keys, values: [pages][heads][tile]
    void* rows[2];                  // [tokens][heads * head_dim] (source, or destination when read)
    long stride[2];                 // elements between rows
    const int* slots;
    int n_tokens, heads, head_dim, groups, page_size, num_pages;
    int* status;
};

template <typename T> __device__ __forceinline__ void load8(const T* p, bool wide, float (&x)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, bool wide, float (&x)[8]) {
    if (wide) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, bool wide, float (&x)[8]) {
    if (wide) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __bfloat162float(p[i]);
    }
}

__device__ __forceinline__ uint32_t code_of(float x, float middle, float step, float inverse) {
    const float d = x - middle;
    const float q = d * inverse;
    float n = rintf(q);
    if (fabsf(fabsf(q - n) - 0.5f) < 1e-4f) {
        const float low = floorf(q);
        float e = fmaf(-(low + 0.5f), step, d);
        if (e == 0.0f) {
            // what x - middle lost when it was rounded (the two sums of Knuth)
            const float t = d - x;
            e = (x - (d - t)) + (-middle - t);
        }
        const bool even = (static_cast<int>(low) & 1) == 0;
        n = e > 0.0f || (e == 0.0f && !even) ? low + 1.0f : low;
    }
    return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(n, -8.0f), 7.0f)) + 8);
}

// The slot of a token, or -1: it has none (recorded where it lies outside the pool).
__device__ __forceinline__ int slot_of(const RowArgs& a, int token) {
    const int slot = a.slots[token];
    if (slot < a.num_pages * a.page_size) return slot;
    if (threadIdx.x == 0 && blockIdx.y == 0) prb_set_status(a.status, PRB_S_SLOT_RANGE, token, slot, a.num_pages);
    return -1;
}

// (Several tokens a CTA, all asked for first, measured no faster for keys coming in and slower for those going back.)
template <typename T>
__global__ void __launch_bounds__(256) kv_append_4bit_kernel(RowArgs a, int wide) {
    prb_grid_launch_dependents();
    prb_grid_wait();
    const int token = blockIdx.x, slot = slot_of(a, token);
    if (slot < 0) return;                               // (the whole CTA)
    const int per = a.heads * a.groups;                 // groups of a token's keys (and of its values)
    const int quarter = threadIdx.x & 3;
    const int unit = (blockIdx.y * blockDim.x + threadIdx.x) >> 2;
    const bool live = unit < 2 * per;
    const int kind = live && unit >= per ? 1 : 0;
    const int hg = live ? unit - kind * per : 0;
    const int head = hg / a.groups, g = hg - head * a.groups;
    const int channel = g * GROUP + quarter * 8;
    const bool has = live && channel < a.head_dim;      // (the last group may be short)
    float x[8];
    float lo = INFINITY, hi = -INFINITY;
    bool fine = true;
    if (has) {
        load8<T>(reinterpret_cast<const T*>(kind ? a.rows[1] : a.rows[0]) + token * (kind ? a.stride[1] : a.stride[0]) +
                     head * a.head_dim + channel,
                 wide != 0, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
            fine = fine && fabsf(x[i]) <= 3.402823466e38f;
        }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const unsigned bad = __ballot_sync(0xffffffffu, !fine);
    if (!has) return;
    fine = ((bad >> (threadIdx.x & 28)) & 15u) == 0;
    // (two roundings, to 32 bits and to bfloat16, as a conversion from 64 bits goes)
    __nv_bfloat16 step_b = __float2bfloat16_rn((float)(((double)hi - (double)lo) / 15.0));
    if (__bfloat162float(step_b) < 1.17549435e-38f) step_b = __float2bfloat16_rn(0.0f);
    const float step = __bfloat162float(step_b);
    __nv_bfloat16 middle_b = __float2bfloat16_rn((float)((double)lo + 8.0 * (double)step));
    const float middle = __bfloat162float(middle_b);
    const float inverse = step > 0.0f ? 1.0f / step : 0.0f;
    uint32_t word = 0;
    if (fine) {
#pragma unroll
        for (int i = 0; i < 8; ++i) word |= code_of(x[i], middle, step, inverse) << (4 * i);
    }
    const int page = slot / a.page_size, at = slot - page * a.page_size;
    uint8_t* tile = (kind ? a.tiles[1] : a.tiles[0]) +
                    ((size_t)page * a.heads + head) * (size_t)cache4::tile_bytes(a.head_dim, a.page_size);
    *reinterpret_cast<uint32_t*>(tile + cache4::code_word(a.head_dim, a.page_size, at, channel / 8)) = word;
    if (quarter == 0) {
        uint32_t pair = (uint32_t)__bfloat16_as_ushort(step_b) | ((uint32_t)__bfloat16_as_ushort(middle_b) << 16);
        if (!fine) pair = 0x7fc07fc0u;
        *reinterpret_cast<uint32_t*>(tile + a.page_size * (a.head_dim / 2) + (at * a.groups + g) * 4) = pair;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) kv_read_4bit_kernel(RowArgs a, int wide) {
    prb_grid_launch_dependents();
    prb_grid_wait();
    const int token = blockIdx.x, slot = slot_of(a, token);
    if (slot < 0) return;
    const int words = a.head_dim / 8, per = a.heads * words;
    const int unit = blockIdx.y * blockDim.x + threadIdx.x;
    if (unit >= 2 * per) return;
    const int page = slot / a.page_size, at = slot - page * a.page_size;
    const int kind = unit >= per ? 1 : 0, hw = unit - kind * per;
    const int head = hw / words, w = hw - head * words;
    const uint8_t* tile = (kind ? a.tiles[1] : a.tiles[0]) +
                          ((size_t)page * a.heads + head) * (size_t)cache4::tile_bytes(a.head_dim, a.page_size);
    const uint32_t word = *reinterpret_cast<const uint32_t*>(tile + cache4::code_word(a.head_dim, a.page_size, at, w));
    const uint32_t pair = *reinterpret_cast<const uint32_t*>(
        tile + a.page_size * (a.head_dim / 2) + (at * a.groups + w / 4) * 4);
    const float step = __uint_as_float(pair << 16), middle = __uint_as_float(pair & 0xffff0000u);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf(step, (float)((int)((word >> (4 * i)) & 15u) - 8), middle);
    T* out = reinterpret_cast<T*>(kind ? a.rows[1] : a.rows[0]) + token * (kind ? a.stride[1] : a.stride[0]) +
             head * a.head_dim + w * 8;
    if (wide) {
        prb_store4(out, x[0], x[1], x[2], x[3]);
        prb_store4(out + 4, x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = prb_from_float<T>(x[i]);
    }
}

int launch_rows(bool append, RowArgs a, int dtype, cudaStream_t stream) {
    if (a.n_tokens <= 0) return 0;
    if (a.heads <= 0 || a.num_pages <= 0 || !cache4::takes(a.head_dim, a.page_size)) return PRB_E_SIZE;
    if ((long)a.num_pages * a.page_size > 0x7fffffffL) return PRB_E_SIZE;
    if (dtype != PRB_F32 && dtype != PRB_BF16) return PRB_E_DTYPE;
    const int size = dtype == PRB_F32 ? 4 : 2;
    bool wide = true;
    for (int i = 0; i < 2; ++i) {
        if ((uintptr_t)a.tiles[i] % 16 != 0) return PRB_E_ALIGN;
        wide = wide && (uintptr_t)a.rows[i] % 16 == 0 && (a.stride[i] * size) % 16 == 0;
    }
    const long pool = a.num_pages * (long)a.heads * cache4::tile_bytes(a.head_dim, a.page_size);
    const long width = (long)a.heads * a.head_dim * size, word = sizeof(int);
    const PrbRange keys{a.tiles[0], pool}, values{a.tiles[1], pool}, slots{a.slots, a.n_tokens * word}, status{a.status, 4 * word};
    const PrbRange k{a.rows[0], prb_span(a.n_tokens, a.stride[0] * size, width)};
    const PrbRange v{a.rows[1], prb_span(a.n_tokens, a.stride[1] * size, width)};
    if (append ? !prb_apart({keys, values, status}, {k, v, slots})
               : !prb_rows_apart(a.rows[0], a.stride[0] * size, a.rows[1], a.stride[1] * size, a.n_tokens, width) ||
                     !prb_apart({k, status}, {keys, values, slots}) || !prb_apart({v, status}, {keys, values, slots}))
        return PRB_E_OVERLAP;
    a.groups = cache4::groups_of(a.head_dim);
    const int threads_of_token = append ? 2 * a.heads * a.groups * 4 : 2 * a.heads * (a.head_dim / 8);
    // (as few CTAs a token as its threads need, of equal size)
    const int blocks = (threads_of_token + 255) / 256, threads = ((threads_of_token + blocks - 1) / blocks + 31) / 32 * 32;
    const dim3 grid(a.n_tokens, blocks);
    cudaError_t e;
    if (append)
        e = dtype == PRB_F32
                ? prb_launch_dependent(kv_append_4bit_kernel<float>, grid, dim3(threads), 0, stream, a, (int)wide)
                : prb_launch_dependent(kv_append_4bit_kernel<__nv_bfloat16>, grid, dim3(threads), 0, stream, a, (int)wide);
    else
        e = dtype == PRB_F32
                ? prb_launch_dependent(kv_read_4bit_kernel<float>, grid, dim3(threads), 0, stream, a, (int)wide)
                : prb_launch_dependent(kv_read_4bit_kernel<__nv_bfloat16>, grid, dim3(threads), 0, stream, a, (int)wide);
    return e == cudaSuccess ? 0 : (int)e;
}
}  // namespace

PRB_API int prb_kv_append_4bit(void* k_tiles, void* v_tiles, const void* k, long k_stride, const void* v, long v_stride,
                               const int* slots, int n_tokens, int kv_heads, int head_dim, int page_size,
                               int num_pages, int dtype, int* status, cudaStream_t stream) {
    RowArgs a{{(uint8_t*)k_tiles, (uint8_t*)v_tiles}, {const_cast<void*>(k), const_cast<void*>(v)}, {k_stride, v_stride},
              slots, n_tokens, kv_heads, head_dim, 0, page_size, num_pages, status};
    return launch_rows(true, a, dtype, stream);
}

PRB_API int prb_kv_read_4bit(void* k_out, long k_stride, void* v_out, long v_stride, const void* k_tiles,
                             const void* v_tiles, const int* slots, int n_tokens, int kv_heads, int head_dim,
                             int page_size, int num_pages, int dtype, int* status, cudaStream_t stream) {
    RowArgs a{{(uint8_t*)const_cast<void*>(k_tiles), (uint8_t*)const_cast<void*>(v_tiles)}, {k_out, v_out},
              {k_stride, v_stride}, slots, n_tokens, kv_heads, head_dim, 0, page_size, num_pages, status};
    return launch_rows(false, a, dtype, stream);
}
