// The cache in 8 bits: e4m3 codes (sign, 4 bits of exponent, 3 of fraction, up to 448; no infinity) and a 32-bit scale, a power
// of two, for each block of 16 positions and key/value head; an entry is code * scale.
//   pages   [pages, kv_heads, page, size] bytes, page and size multiples of 16
//   scales  [pages, kv_heads, page / 16] fp32
// A head's positions of a page lie side by side, so that a block is one contiguous piece of 16 * size bytes.
#pragma once

#include <limits.h>

#include <atomic>

#include "common.cuh"

constexpr int E4M3_BLOCK = 16;                 // positions that share a scale
constexpr int E4M3_LEAST_EXPONENT = -64;       // of a scale

// Two numbers to two codes, nearest, ties to even; beyond 448 to 448, what is no number to the code that is none.
__device__ __forceinline__ uint32_t e4m3_pair(float low, float high) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(high), "f"(low));
    return r;
}

// Two codes to two 16-bit floats (every code is one exactly).
__device__ __forceinline__ uint32_t e4m3_to_half2(uint16_t pair) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(pair));
    return r;
}
__device__ __forceinline__ void e4m3_to_half2(uint32_t four, uint32_t& low, uint32_t& high) {
    low = e4m3_to_half2((uint16_t)(four & 0xffffu));
    high = e4m3_to_half2((uint16_t)(four >> 16));
}

__device__ __forceinline__ float2 half2_to_floats(uint32_t h) {
    float2 r;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(h));
    return r;
}

// Two numbers to two 16-bit floats, nearest.
__device__ __forceinline__ uint32_t half2_of(float low, float high) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
    return r;
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }     // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float power) { return ((__float_as_int(power) >> 23) & 255) - 127; }

// 2^x by the hardware (about 2 ulp).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Queries as 16-bit floats: the e for which 2^e brings the largest entry of a head to between 2^14 and 2^15.  From -113 on, for entries up to 2^128; not beyond
// 110, whose inverse and scale still make a number (entries below 2^-96 become smaller ones).  Zeros, and what is not finite, stay as they are.
__device__ __forceinline__ int query_exponent(float largest) {
    return largest > 0.0f && largest < INFINITY ? min(110, 14 - exponent_of(largest)) : 0;
}
// What brings a head's scores into place as a number: an infinite one would make none of a product of zero.  Where it is cut off, at 2^128, scores differ by
// 2^30 and more or not at all (a product is a whole number of 2^-33, a key's scale 2^-64 or more), and do so still.  (Cutting it off again where it
// meets a block's scale, in the loops, cost 3 % of a long prompt and 5 % of 64 single tokens; what the caller keeps to excludes that it passes 2^128 there.)
__device__ __forceinline__ float finite_factor(float factor) { return fminf(factor, 3.402823466e38f); }

// a / b of numbers that are not negative (the 64-bit division costs some hundred clocks, and a row is hardly ever that long).
__device__ __forceinline__ long divided(long a, long b) {
    return ((a | b) >> 31) == 0 ? (long)((uint32_t)a / (uint32_t)b) : a / b;
}

// cap * tanh(x / cap) = cap * (1 - 2 / (1 + e^(2x / cap))): two of the hardware's approximations with an error of some 2^-22 of the
// cap, where its approximate tanh has 2^-11: of a cap of 50 that would be 2.4 % of a weight.
__device__ __forceinline__ float capped(float x, float cap, float two_log2e_over_cap) {
    const float e = exp2_fast(x * two_log2e_over_cap);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return cap - 2.0f * cap * r;
}

// Raises a kernel's limit of dynamic shared memory, once on each device (`raised`), to the `most` that any launch of it takes: threads that come here at the
// same time set the same limit, whatever the sizes of their calls.
template <typename Kernel>
static cudaError_t raise_shared_limit(Kernel kernel, size_t most, std::atomic<bool> (&raised)[64]) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 64 && raised[device])) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e == cudaSuccess && device < 64) raised[device] = true;
    return e;
}

// What storing gets.
struct E4m3Store {
    void* q_out;                   // [n, heads * dim] or null: the queries stay as they are
    long ld_q;
    const void* qkv;
    long ld;
    int k_off, v_off, heads, kv_heads, dim, vdim, rot_dims;
    const double* inv_freq;
    float amplitude;
    const int *positions, *token_item, *block_table;
    int max_blocks, n_pages, page;
    uint8_t *k_pages, *v_pages;    // null: nothing is stored
    float *k_scales, *v_scales;
    int n;
};
static_assert(sizeof(E4m3Store) == 160, "packed by the caller field by field, with C's alignment");

// What attention over the cache gets.  An entry is a request's tokens of this step: rows item_offset .. + item_count of q, at
// positions item_start, item_start + 1, ...; entries without tokens are allowed.
struct E4m3Attention {
    void* out;                     // [rows, heads * vdim]
    long ld_out;
    const void* q;                 // [rows, heads * dim]
    long ld_q;
    const uint8_t *k_pages, *v_pages;
    const float *k_scales, *v_scales;
    const int* block_table;        // [entries, max_blocks]
    int max_blocks, n_pages, page;
    const int *item_offset, *item_count, *item_start;
    int n_items;
    int n_heads, n_kv_heads, dim, vdim;
    float scale, cap;              // cap 0: none
    int window;                    // 0: all keys
    float* partial;                // results of parts, and how many of a result's parts have arrived (zero between launches)
    int* counters;
    int* status;                   // where a bounded wait that ran out leaves its code
    int wait_limit_ns;             // of every wait; 0: as elsewhere
    int role_away;                 // a test's switch: the role with this give-up code does nothing, and the others' waits run out; 0: none
};
static_assert(sizeof(E4m3Attention) == 176, "packed by the caller field by field, with C's alignment");

// The keys that a query at a position sees: from here on (within a window, which may be as long as an int; positions may lie before the first) ...
__device__ __forceinline__ int first_seen(int position, int window) { return window > 0 && position >= window ? position - window + 1 : 0; }
// ... up to its own, but for those behind the last that a request's row of the block table names, where every walk ends (a row of blocks of 128 from there
// on is counted in an int).
__device__ __forceinline__ int last_seen(int position, const E4m3Attention& p) {
    return (int)min((long)position, min((long)p.max_blocks * p.page, (long)INT_MAX - 255) - 1);
}
