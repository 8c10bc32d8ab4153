// The 8-bit cache (e4m3.cuh): storing a step's keys and values, with the rotation of queries and keys on the way, and attention
// over it for single tokens (mma.sync tiles) and, as a plain twin for every size and type, for any row.
#include "common.cuh"
#include "e4m3.cuh"

MLLM_DEFINE_ERROR_API(mllm_e4m3)

namespace {

// ---- storing ------------------------------------------------------------------------------------
//
// The scale of a block is the least power of two s >= 2^-64 with n <= (448 s)^2 for all its rows, n the square of the length
// of a pair that turns (which the turn keeps) and of any other entry.  It is known before any angle, and from 16-bit
// inputs the same bit for bit whoever computes it: their squares are exact, and a sum of two is rounded once.  Being a power of two
// it moves codes without rounding them (but for the smallest, which lie below the code's normal range), when a row that joins a block
// raises it.  A row in which some n is not finite (an infinity, no number, or beyond 2^64) is stored as no number throughout, since e4m3
// has no infinity, and does not count.
//
// A block of 16 positions belongs to the warp that has its first row of this step ("leader"): it reads the rows of the block, takes the
// maximum, raises the codes that are there already where it must, and writes the new ones: no two warps touch a block, and
// a step that is run again leaves the same bytes.  A CTA takes G rows and the blocks that begin in them, and a share of the heads; its
// table of cosines and sines serves all of them (an angle per head cost 22 of 28 us for 8,192 tokens of 40 turned heads of 96 by
// its instruction count).  What bounds it is bytes: rows once in, codes and queries once out.
struct StoreParams {
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

constexpr int STORE_THREADS = 256, STORE_ROWS = 16;

// Eight numbers of a row.
__device__ __forceinline__ void load_eight(const bf16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ void load_eight(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void store_eight(bf16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_eight(float* p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

// The pairs of columns `first` .. + 7 that lie among the turned ones.
__device__ __forceinline__ void turn_eight(float (&x)[8], int first, int rot_dims, const float2* angles) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (first + 2 * i < rot_dims) {
            const float2 a = angles[first / 2 + i];
            const float u = x[2 * i] * a.x - x[2 * i + 1] * a.y, v = x[2 * i] * a.y + x[2 * i + 1] * a.x;
            x[2 * i] = u, x[2 * i + 1] = v;
        }
    }
}

// The largest square of eight columns, as bits: what is no number, or no finite one, is the largest of all.
__device__ __forceinline__ uint32_t square_bits(const float (&x)[8], int first, int rot_dims, float amplitude_squared) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = __fmul_rn(x[2 * i], x[2 * i]), b = __fmul_rn(x[2 * i + 1], x[2 * i + 1]);
        if (first + 2 * i < rot_dims) {
            most = max(most, __float_as_uint(__fmul_rn(__fadd_rn(a, b), amplitude_squared)));
        } else {
            most = max(most, max(__float_as_uint(a), __float_as_uint(b)));
        }
    }
    return most;
}

// The least e >= -64 with square <= (448 * 2^e)^2.
__device__ __forceinline__ int scale_exponent(float square) {
    // square = m 2^x, m in [1, 2), and 448^2 = 1.53125 * 2^17
    const int bits = __float_as_int(square), x = (bits >> 23) - 127;
    const int twice = x - 17 + ((bits & 0x7fffff) > 0x440000 ? 1 : 0);          // 4^e must reach 2^twice
    return max((twice + 1) >> 1, E4M3_LEAST_EXPONENT);
}

template <typename T>
__global__ void __launch_bounds__(STORE_THREADS) store_kernel(const StoreParams p, int G) {
    __shared__ int row_pos[STORE_ROWS + 16], row_item[STORE_ROWS + 16];        // of rows first - 1, first, ...
    extern __shared__ float2 angles[];                                         // [rows, rot_dims / 2]
    dependents_may_start();
    const int first = blockIdx.x * G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int most = min(G + 15, p.n - first);         // the rows that may matter: a block that begins in the last row has 15 more
    const int own_rows = min(G, p.n - first);
    wait_for_earlier_kernels();
    if ((int)threadIdx.x <= most) {
        const int row = first - 1 + threadIdx.x;
        row_pos[threadIdx.x] = row >= 0 ? p.positions[row] : -2;
        row_item[threadIdx.x] = row >= 0 ? p.token_item[row] : -1;
    }
    __syncthreads();
    // A row leads where it does not go on in the block of the row before it.
    uint32_t leads = 0;
    {
        bool lead = true;
        if (lane < most) {
            const int pos = row_pos[lane + 1];
            lead = row_item[lane] != row_item[lane + 1] || row_pos[lane] + 1 != pos || (pos & (E4M3_BLOCK - 1)) == 0 || pos < 0;
        }
        leads = __ballot_sync(0xffffffffu, lead);                              // (rows behind the last one: all)
    }
    const uint32_t mine = own_rows < 32 ? (1u << own_rows) - 1u : 0xffffffffu;
    int rows = own_rows;                                                       // rows whose angles are needed
    if (p.k_pages != nullptr && (leads & mine) != 0) {
        const uint32_t behind = leads >> own_rows;                             // (own_rows <= 16 < 32)
        rows = min(most, own_rows + (behind != 0 ? __ffs(behind) - 1 : 31));
    }
    const int half = p.rot_dims / 2;
    for (int i = threadIdx.x; i < rows * half; i += STORE_THREADS) {
        const int r = i / half;
        // the angle in turns, 64-bit until less than one of them is left
        double turns = (double)row_pos[r + 1] * p.inv_freq[i - r * half] * 0.15915494309189535;
        turns -= rint(turns);
        float s, c;
        sincospif((float)(2.0 * turns), &s, &c);
        angles[i] = make_float2(c * p.amplitude, s * p.amplitude);
    }
    __syncthreads();
    const T* qkv = behind_the_wait(static_cast<const T*>(p.qkv));
    const int q_slots = p.q_out != nullptr ? p.heads : 0;
    const int slots = q_slots + (p.k_pages != nullptr ? 2 * p.kv_heads : 0);
    const int stride = gridDim.y * (STORE_THREADS / 32);
    for (int slot = blockIdx.y * (STORE_THREADS / 32) + warp; slot < slots; slot += stride) {
        if (slot < q_slots) {
            const int chunks = p.dim / 8;
#pragma unroll 4
            for (int u = lane; u < own_rows * chunks; u += 32) {
                const int r = u / chunks, col = (u - r * chunks) * 8;
                float x[8];
                load_eight(qkv + (first + r) * p.ld + (long)slot * p.dim + col, x);
                turn_eight(x, col, p.rot_dims, angles + r * half);
                store_eight(static_cast<T*>(p.q_out) + (first + r) * p.ld_q + (long)slot * p.dim + col, x);
            }
            continue;
        }
        const bool values = slot >= q_slots + p.kv_heads;
        const int head = slot - q_slots - (values ? p.kv_heads : 0);
        const int size = values ? p.vdim : p.dim, rot = values ? 0 : p.rot_dims, chunks = size / 8;
        const float amplitude_squared = p.amplitude * p.amplitude;
        const T* from = qkv + (values ? p.v_off : p.k_off) + (long)head * size;
        uint8_t* pages = values ? p.v_pages : p.k_pages;
        float* scales = values ? p.v_scales : p.k_scales;
        for (uint32_t todo = leads & mine; todo != 0; todo &= todo - 1) {
            const int r0 = __ffs(todo) - 1;
            const uint32_t after = leads >> (r0 + 1);                          // (r0 <= 15)
            const int count = min(after != 0 ? __ffs(after) : 32, most - r0);
            const int pos = row_pos[r0 + 1], item = row_item[r0 + 1];
            const int index = pos >= 0 ? pos / p.page : p.max_blocks;
            if (index >= p.max_blocks) continue;
            const int page_id = p.block_table[(long)item * p.max_blocks + index];
            if (page_id < 0 || page_id >= p.n_pages) continue;
            const int slot0 = pos - index * p.page, lead = pos & (E4M3_BLOCK - 1);
            const long place = (long)page_id * p.kv_heads + head;
            float* scale_at = scales + place * (p.page / E4M3_BLOCK) + slot0 / E4M3_BLOCK;
            const float held = lead > 0 ? *scale_at : 0.0f;
            uint32_t top = 0;
#pragma unroll 4
            for (int u = lane; u < count * chunks; u += 32) {
                const int r = u / chunks, col = (u - r * chunks) * 8;
                float x[8];
                load_eight(from + (first + r0 + r) * p.ld + col, x);
                top = max(top, square_bits(x, col, rot, amplitude_squared));
            }
            top = __reduce_max_sync(0xffffffffu, top);
            uint32_t bad = 0;                                                  // rows that are not finite
            if (top >= 0x7f800000u) {
                top = 0;
                for (int r = 0; r < count; r++) {
                    uint32_t of_row = 0;
                    for (int col = lane * 8; col < size; col += 256) {
                        float x[8];
                        load_eight(from + (first + r0 + r) * p.ld + col, x);
                        of_row = max(of_row, square_bits(x, col, rot, amplitude_squared));
                    }
                    of_row = __reduce_max_sync(0xffffffffu, of_row);
                    if (of_row >= 0x7f800000u) bad |= 1u << r;
                    else top = max(top, of_row);
                }
            }
            const float needed = power_of_two(scale_exponent(__uint_as_float(top)));
            const float scale = fmaxf(held, needed);
            uint8_t* block = pages + (place * p.page + slot0 - lead) * size;
            if (lead > 0 && scale > held) {
                const float down = held / scale;                               // powers of two
                for (int u = lane; u < lead * (size / 16); u += 32) {
                    uint4 v = reinterpret_cast<const uint4*>(block)[u];
                    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t low, high;
                        e4m3_to_half2(w[i], low, high);
                        const float2 a = half2_to_floats(low), b = half2_to_floats(high);
                        w[i] = e4m3_pair(a.x * down, a.y * down) | (e4m3_pair(b.x * down, b.y * down) << 16);
                    }
                    reinterpret_cast<uint4*>(block)[u] = v;
                }
            }
            if (lane == 0 && scale != held) *scale_at = scale;
            const float inverse = 1.0f / scale;
#pragma unroll 4
            for (int u = lane; u < count * chunks; u += 32) {
                const int r = u / chunks, col = (u - r * chunks) * 8;
                float x[8];
                load_eight(from + (first + r0 + r) * p.ld + col, x);
                turn_eight(x, col, rot, angles + (r0 + r) * half);
                uint2 codes;
                codes.x = e4m3_pair(x[0] * inverse, x[1] * inverse) | (e4m3_pair(x[2] * inverse, x[3] * inverse) << 16);
                codes.y = e4m3_pair(x[4] * inverse, x[5] * inverse) | (e4m3_pair(x[6] * inverse, x[7] * inverse) << 16);
                if ((bad >> r) & 1) codes = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
                *reinterpret_cast<uint2*>(block + (long)(lead + r) * size + col) = codes;
            }
        }
    }
}

// ---- attention, plain ---------------------------------------------------------------------------
//
// A CTA takes a row and a head: 128 keys at a time, a thread a key's score, then a thread a column of the values.  All in 32 bits.
constexpr int PLAIN_THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(PLAIN_THREADS) attention_plain_kernel(const E4m3Attention p) {
    __shared__ float q[256], weight[PLAIN_THREADS], scratch[PLAIN_THREADS / 32];
    __shared__ long place[PLAIN_THREADS];                // of the 128 keys: (page * kv_heads + head) * page size + slot, or -1
    __shared__ int entry;
    dependents_may_start();
    wait_for_earlier_kernels();
    const int row = blockIdx.x, head = blockIdx.y, kv_head = head / (p.n_heads / p.n_kv_heads);
    if (threadIdx.x == 0) entry = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < p.n_items; i += PLAIN_THREADS)
        if (row >= p.item_offset[i] && row < p.item_offset[i] + p.item_count[i]) entry = i;
    __syncthreads();
    if (entry < 0) return;                               // rows behind the last entry stay as they are
    const int pos = p.item_start[entry] + row - p.item_offset[entry];
    const int first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    for (int d = threadIdx.x; d < p.dim; d += PLAIN_THREADS)
        q[d] = to_f32(static_cast<const T*>(p.q)[row * p.ld_q + (long)head * p.dim + d]);
    float o[2] = {0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
    for (int base = first; base <= pos; base += PLAIN_THREADS) {
        const int key = base + threadIdx.x, index = key / p.page;
        float s = -INFINITY;
        long at = -1;
        __syncthreads();
        if (key <= pos && index < p.max_blocks) {
            const int id = p.block_table[(long)entry * p.max_blocks + index];
            if (id >= 0 && id < p.n_pages) at = ((long)id * p.n_kv_heads + kv_head) * p.page + key % p.page;
        }
        if (at >= 0) {
            const uint4* codes = reinterpret_cast<const uint4*>(p.k_pages + at * p.dim);
            float sum = 0.0f;
            for (int c = 0; c < p.dim / 16; c++) {
                const uint4 v = codes[c];
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t low, high;
                    e4m3_to_half2(w[i], low, high);
                    const float2 a = half2_to_floats(low), b = half2_to_floats(high);
                    const float* x = q + 16 * c + 4 * i;
                    sum += x[0] * a.x + x[1] * a.y + x[2] * b.x + x[3] * b.y;
                }
            }
            s = sum * p.k_scales[at / E4M3_BLOCK] * p.scale;
            if (p.cap > 0.0f) s = p.cap * tanhf(s / p.cap);
        }
        place[threadIdx.x] = at;
        const float top = warp_max(s);
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = top;
        __syncthreads();
        const float m_new = fmaxf(fmaxf(m, fmaxf(scratch[0], scratch[1])), fmaxf(scratch[2], scratch[3]));
        const float anchor = m_new == -INFINITY ? 0.0f : m_new, down = expf(m - anchor);
        weight[threadIdx.x] = at >= 0 ? expf(s - anchor) : 0.0f;
        m = m_new;
        __syncthreads();
        float sum = 0.0f;
        o[0] *= down, o[1] *= down;
        for (int k = 0; k < PLAIN_THREADS; k++) {
            const long there = place[k];
            if (there < 0) continue;
            const float w = weight[k], wv = w * p.v_scales[there / E4M3_BLOCK];
            sum += w;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int d = threadIdx.x + i * PLAIN_THREADS;
                if (d < p.vdim) o[i] += wv * half2_to_floats(e4m3_to_half2((uint16_t)p.v_pages[there * p.vdim + d])).x;
            }
        }
        l = l * down + sum;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int d = threadIdx.x + i * PLAIN_THREADS;
        if (d < p.vdim) static_cast<T*>(p.out)[row * p.ld_out + (long)head * p.vdim + d] = from_f32<T>(l == 0.0f ? 0.0f : o[i] / l);
    }
}

// ---- attention of single tokens -----------------------------------------------------------------
//
// The entries of one token.  What bounds them is the cache: every visible code is read once.  A CTA takes a token, a key/value head with
// up to 16 of its query heads, and a part of the keys; its eight warps take the blocks of 16 keys in turn.  A warp reads a block straight into
// registers in the layout of mma.sync m16n8k16, the codes as 16-bit floats (each is one exactly):
//   S = Q K^T: key g (of 8) and columns 16 c .. 16 c + 15 of it lie with lane 4 g + c: one load of 16 bytes, four products; the order of
//     the columns within a product does not matter as long as Q has the same;
//   O = P V: keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 and columns 8 g .. 8 g + 7 of each: the pairs of keys are put together byte by byte.
// Q is scaled by a power of two to lie below 2^15 in 16-bit floats (11 bits: bfloat16's 8 fit; an entry 2^29 below the largest of its head
// begins to lose some, where the 32-bit sum has lost it already).  The weights: a block's value scale 2^t joins the score as t in
// the exponent, p = 2^(s + t - m + 7), and the sum of the weights gets p / 2^t: no multiplication more, and p keeps the 11 bits of a 16-bit
// float however far apart the scales lie.  m moves only where a score passes it by 8, so that p stays below 2^15.
constexpr int STEP_WARPS = 8, STEP_THREADS = STEP_WARPS * 32;
constexpr int STEP_MIN_BLOCKS = 8;             // a part has a block of keys at least for every warp

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same where rows 8 to 15 are empty: their sums are not kept.
__device__ __forceinline__ void mma_f16_upper(float& c0, float& c1, uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
    [[maybe_unused]] float none0, none1;
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %6, %5, %6}, {%7, %8}, {%0, %1, %9, %9};"
                 : "+f"(c0), "+f"(c1), "=f"(none0), "=f"(none1)
                 : "r"(a0), "r"(a2), "r"(0u), "r"(b0), "r"(b1), "f"(0.0f));
}

// KG, VG: groups of 64 columns of a key and a value; HALVES 1: at most eight query heads, 2: sixteen.
template <int KG, int VG, int HALVES>
__global__ void __launch_bounds__(STEP_THREADS, HALVES * VG <= 2 ? 2 : 1) attention_step_kernel(const E4m3Attention p, int head_tiles, int max_parts) {
    extern __shared__ float shared[];
    __shared__ int ticket;
    dependents_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int entry = blockIdx.z, kv_head = blockIdx.y / head_tiles, head_tile = blockIdx.y % head_tiles, part = blockIdx.x;
    const int group = p.n_heads / p.n_kv_heads;
    const int n_rows = min(8 * HALVES, group - head_tile * 8 * HALVES);
    const int head0 = kv_head * group + head_tile * 8 * HALVES;
    wait_for_earlier_kernels();
    if (p.item_count[entry] != 1) return;
    const int row = p.item_offset[entry], pos = p.item_start[entry];
    const int first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    const int block_lo = first / E4M3_BLOCK;
    const int n_blocks = pos >= 0 ? min(pos / E4M3_BLOCK + 1, p.max_blocks * (p.page / E4M3_BLOCK)) - block_lo : 0;
    const int per_part = max(STEP_MIN_BLOCKS, (n_blocks + max_parts - 1) / max_parts);
    const int n_parts = max(1, (n_blocks + per_part - 1) / per_part);
    if (part >= n_parts) return;
    const int lo = block_lo + part * per_part, hi = min(lo + per_part, block_lo + n_blocks);

    // the queries, as 16-bit floats of a power of two's size, in the order of the key's columns (in shared memory: all warps have the same)
    const bf16* q = static_cast<const bf16*>(p.q) + row * p.ld_q;
    __shared__ uint4 qa[HALVES][KG][2][32];
    float q_factor[HALVES];                      // what brings a score into powers of two
#pragma unroll
    for (int h = 0; h < HALVES; h++) {
        const int r = g + 8 * h;
        float x[KG][16], top = 0.0f;
#pragma unroll
        for (int d = 0; d < KG; d++) {
            const int col = 64 * d + 16 * c;
#pragma unroll
            for (int i = 0; i < 16; i++) x[d][i] = 0.0f;
            if (r < n_rows && col < p.dim) {
                const uint4* at = reinterpret_cast<const uint4*>(q + (long)(head0 + r) * p.dim + col);
                const uint4 u = at[0], v = at[1];
                const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 8; i++) x[d][2 * i] = __uint_as_float(w[i] << 16), x[d][2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, fabsf(x[d][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // (zeros, and what is not finite, stay as they are)
        const int e = top > 0.0f && top < INFINITY ? max(-110, min(110, 14 - exponent_of(top))) : 0;
        const float factor = power_of_two(e);
        q_factor[h] = p.scale * power_of_two(-e);
        if (warp == 0)
#pragma unroll
            for (int d = 0; d < KG; d++)
#pragma unroll
                for (int s = 0; s < 2; s++)
                    qa[h][d][s][lane] = make_uint4(half2_of(x[d][8 * s] * factor, x[d][8 * s + 1] * factor),
                                                   half2_of(x[d][8 * s + 2] * factor, x[d][8 * s + 3] * factor),
                                                   half2_of(x[d][8 * s + 4] * factor, x[d][8 * s + 5] * factor),
                                                   half2_of(x[d][8 * s + 6] * factor, x[d][8 * s + 7] * factor));
    }
    __syncthreads();
    constexpr float LOG2E = 1.4426950408889634f;
    const bool has_cap = p.cap > 0.0f;
    if (!has_cap)
        for (int h = 0; h < HALVES; h++) q_factor[h] *= LOG2E;
    const float cap_factor = has_cap ? 2.0f * LOG2E / p.cap : 0.0f, cap_log2 = p.cap * LOG2E;

    float acc[VG][8][2 * HALVES], m[HALVES], l[HALVES];
#pragma unroll
    for (int d = 0; d < VG; d++)
#pragma unroll
        for (int t = 0; t < 8; t++)
#pragma unroll
            for (int i = 0; i < 2 * HALVES; i++) acc[d][t][i] = 0.0f;
#pragma unroll
    for (int h = 0; h < HALVES; h++) m[h] = -INFINITY, l[h] = 0.0f;

    const int per_page = p.page / E4M3_BLOCK;
    const int* table = p.block_table + (long)entry * p.max_blocks;
    const uint8_t* k_pages = behind_the_wait(p.k_pages);
    const uint8_t* v_pages = behind_the_wait(p.v_pages);
    // Lane i looks up the warp's next 32 blocks: where block i lies (in blocks), and its scales.
    long of_lane = -1;
    float k_scale_of_lane = 0.0f, v_scale_of_lane = 0.0f;
    auto look_up = [&](int from) {
        const int b = from + lane * STEP_WARPS;
        of_lane = -1;
        if (b < hi) {
            const int id = table[b / per_page];
            if (id >= 0 && id < p.n_pages) {
                of_lane = ((long)id * p.n_kv_heads + kv_head) * per_page + b % per_page;
                k_scale_of_lane = p.k_scales[of_lane];
                v_scale_of_lane = p.v_scales[of_lane];
            }
        }
    };
    struct Block {
        uint4 k[2][KG];
        uint2 v[4][VG];
        float k_scale, v_scale;
        bool there;
    };
    auto fetch = [&](Block& b, int i) {                  // the i-th of the blocks that were looked up
        const long at = __shfl_sync(0xffffffffu, of_lane, i);
        b.k_scale = __shfl_sync(0xffffffffu, k_scale_of_lane, i);
        b.v_scale = __shfl_sync(0xffffffffu, v_scale_of_lane, i);
        b.there = at >= 0;
        const uint8_t* k = k_pages + at * E4M3_BLOCK * p.dim;
        const uint8_t* v = v_pages + at * E4M3_BLOCK * p.vdim;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int d = 0; d < KG; d++) {
                const int col = 64 * d + 16 * c;
                b.k[h][d] = make_uint4(0u, 0u, 0u, 0u);
                if (b.there && col < p.dim) b.k[h][d] = __ldcs(reinterpret_cast<const uint4*>(k + (8 * h + g) * p.dim + col));
            }
#pragma unroll
        for (int i4 = 0; i4 < 4; i4++)
#pragma unroll
            for (int d = 0; d < VG; d++) {
                const int col = 64 * d + 8 * g, key = 2 * c + (i4 & 1) + 8 * (i4 >> 1);
                b.v[i4][d] = make_uint2(0u, 0u);
                if (b.there && col < p.vdim) b.v[i4][d] = __ldcs(reinterpret_cast<const uint2*>(v + key * p.vdim + col));
            }
    };
    auto work = [&](Block& b, int index) {
        if (!b.there) return;
        float s[2][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            s[h][0] = s[h][1] = s[h][2] = s[h][3] = 0.0f;
#pragma unroll
            for (int d = 0; d < KG; d++) {
                const uint32_t w[4] = {b.k[h][d].x, b.k[h][d].y, b.k[h][d].z, b.k[h][d].w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint4 lower = qa[0][d][i >> 1][lane], upper = qa[HALVES - 1][d][i >> 1][lane];
                    uint32_t b0, b1;
                    e4m3_to_half2(w[i], b0, b1);
                    if (HALVES == 1) mma_f16_upper(s[h][0], s[h][1], (i & 1) ? lower.z : lower.x, (i & 1) ? lower.w : lower.y, b0, b1);
                    else mma_f16(s[h], (i & 1) ? lower.z : lower.x, (i & 1) ? upper.z : upper.x, (i & 1) ? lower.w : lower.y, (i & 1) ? upper.w : upper.y, b0, b1);
                }
            }
        }
        const float t = (float)exponent_of(b.v_scale), over = 1.0f / b.v_scale;
        const int key0 = index * E4M3_BLOCK;
        const bool partial = key0 + E4M3_BLOCK - 1 > pos || key0 < first;
        // the weights of rows g and g + 8, keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9
        uint32_t pa[HALVES][2];
        float x[HALVES][4], top[HALVES];
        bool moves = false;
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            const float factor = q_factor[h] * b.k_scale;
            top[h] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float y = s[i >> 1][2 * h + (i & 1)] * factor;
                y = has_cap ? capped(y, cap_log2, cap_factor) + t : y + t;
                const int key = key0 + 2 * c + (i & 1) + 8 * (i >> 1);
                if (partial && (key > pos || key < first)) y = -INFINITY;
                x[h][i] = y;
                top[h] = fmaxf(top[h], y);
            }
            moves = moves || top[h] > m[h] + 8.0f;
        }
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                float most = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                most = fmaxf(m[h], fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2)));
                const float down = m[h] == -INFINITY ? 0.0f : exp2_fast(m[h] - most);
                m[h] = most;
                l[h] *= down;
#pragma unroll
                for (int d = 0; d < VG; d++)
#pragma unroll
                    for (int i = 0; i < 8; i++) acc[d][i][2 * h] *= down, acc[d][i][2 * h + 1] *= down;
            }
        }
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            const float base = (m[h] == -INFINITY ? 0.0f : m[h]) - 7.0f;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[h][i] = exp2_fast(x[h][i] - base);
                sum += x[h][i];
            }
            l[h] += sum * over;
            pa[h][0] = half2_of(x[h][0], x[h][1]);
            pa[h][1] = half2_of(x[h][2], x[h][3]);
        }
        if (partial) {
            // a masked key's value may be no number, and its weight of zero would not keep it out
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int key = key0 + 2 * c + (i & 1) + 8 * (i >> 1);
                if (key > pos || key < first)
#pragma unroll
                    for (int d = 0; d < VG; d++) b.v[i][d] = make_uint2(0u, 0u);
            }
        }
#pragma unroll
        for (int d = 0; d < VG; d++)
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const uint32_t v0 = w ? b.v[0][d].y : b.v[0][d].x, v1 = w ? b.v[1][d].y : b.v[1][d].x;
                const uint32_t v2 = w ? b.v[2][d].y : b.v[2][d].x, v3 = w ? b.v[3][d].y : b.v[3][d].x;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    // columns 2 half and 2 half + 1 of the four: (key a, key b) of the one, then of the other
                    const uint32_t order = half ? 0x7362 : 0x5140;
                    uint32_t b00, b01, b10, b11;
                    e4m3_to_half2(__byte_perm(v0, v1, order), b00, b01);
                    e4m3_to_half2(__byte_perm(v2, v3, order), b10, b11);
                    float(&even)[2 * HALVES] = acc[d][4 * w + 2 * half];
                    float(&odd)[2 * HALVES] = acc[d][4 * w + 2 * half + 1];
                    if constexpr (HALVES == 1) {
                        mma_f16_upper(even[0], even[1], pa[0][0], pa[0][1], b00, b10);
                        mma_f16_upper(odd[0], odd[1], pa[0][0], pa[0][1], b01, b11);
                    } else {
                        mma_f16(even, pa[0][0], pa[1][0], pa[0][1], pa[1][1], b00, b10);
                        mma_f16(odd, pa[0][0], pa[1][0], pa[0][1], pa[1][1], b01, b11);
                    }
                }
            }
    };
    // two blocks on their way while one is worked on
    int taken = 0;
    Block a, b;
    const int mine = lo + warp < hi ? (hi - lo - warp + STEP_WARPS - 1) / STEP_WARPS : 0;
    auto next = [&](Block& x) {
        if (taken >= mine) return;
        if ((taken & 31) == 0) look_up(lo + warp + taken * STEP_WARPS);
        fetch(x, taken & 31);
        taken++;
    };
    next(a);
    for (int i = 0; i < mine; i += 2) {
        next(b);
        work(a, lo + warp + i * STEP_WARPS);
        next(a);
        if (i + 1 < mine) work(b, lo + warp + (i + 1) * STEP_WARPS);
    }

    // the warps' results: rows of [vdim] sums, then the maxima and the sums of the weights
    const int width = 64 * VG;
    float* of_m = shared + STEP_WARPS * n_rows * width;
    float* of_l = of_m + STEP_WARPS * n_rows;
#pragma unroll
    for (int h = 0; h < HALVES; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const int r = g + 8 * h;
        // (lanes of a row agree on its maximum, but for rows whose scores never passed a warp's vote)
        if (r < n_rows) {
            if (c == 0) of_m[warp * n_rows + r] = m[h], of_l[warp * n_rows + r] = l[h];
            float* to = shared + (warp * n_rows + r) * width;
#pragma unroll
            for (int d = 0; d < VG; d++)
#pragma unroll
                for (int t = 0; t < 8; t += 4)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        *reinterpret_cast<float4*>(to + 64 * d + 16 * c + 8 * e + t) =
                            make_float4(acc[d][t][2 * h + e], acc[d][t + 1][2 * h + e], acc[d][t + 2][2 * h + e], acc[d][t + 3][2 * h + e]);
        }
    }
    __syncthreads();
    bf16* out = static_cast<bf16*>(p.out) + row * p.ld_out + (long)head0 * p.vdim;
    const int cell = entry * gridDim.y + blockIdx.y, part_floats = 8 * HALVES * (width + 2);
    float* all = p.partial + (long)cell * max_parts * part_floats;
    float* mine_out = all + (long)part * part_floats;
    for (int i = threadIdx.x; i < n_rows * width; i += STEP_THREADS) {
        const int r = i / width, col = i - r * width;
        float top = -INFINITY, sum = 0.0f, total = 0.0f;
#pragma unroll
        for (int w = 0; w < STEP_WARPS; w++) top = fmaxf(top, of_m[w * n_rows + r]);
        const float anchor = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < STEP_WARPS; w++) {
            const float weight = exp2_fast(of_m[w * n_rows + r] - anchor);
            sum += weight * shared[(w * n_rows + r) * width + col];
            total += weight * of_l[w * n_rows + r];
        }
        if (n_parts == 1) {
            if (col < p.vdim) out[r * p.vdim + col] = __float2bfloat16_rn(total == 0.0f ? 0.0f : sum / total);
        } else {
            __stcg(mine_out + i, sum);
            if (col == 0) __stcg(mine_out + 8 * HALVES * width + 2 * r, top), __stcg(mine_out + 8 * HALVES * width + 2 * r + 1, total);
        }
    }
    if (n_parts == 1) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) ticket = atomicAdd(p.counters + cell, 1);
    __syncthreads();
    if (ticket != n_parts - 1) return;
    __threadfence();
    // the last to arrive adds the parts up, in their order
    for (int i = threadIdx.x; i < n_rows * width; i += STEP_THREADS) {
        const int r = i / width, col = i - r * width;
        const float* state = all + 8 * HALVES * width + 2 * r;
        float top = -INFINITY, sum = 0.0f, total = 0.0f;
        for (int q = 0; q < n_parts; q++) top = fmaxf(top, __ldcg(state + (long)q * part_floats));
        const float anchor = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
        for (int q = 0; q < n_parts; q++) {
            const float weight = exp2_fast(__ldcg(state + (long)q * part_floats) - anchor);
            sum += weight * __ldcg(all + (long)q * part_floats + i);
            total += weight * __ldcg(state + (long)q * part_floats + 1);
        }
        if (col < p.vdim) out[r * p.vdim + col] = __float2bfloat16_rn(total == 0.0f ? 0.0f : sum / total);
    }
    if (threadIdx.x == 0) p.counters[cell] = 0;
}

template <int KG, int VG, int HALVES>
int launch_step(const E4m3Attention& p, int n_sms, cudaStream_t stream) {
    const int group = p.n_heads / p.n_kv_heads, rows = min(group, 8 * HALVES);
    const int head_tiles = (group + 8 * HALVES - 1) / (8 * HALVES);
    const long cells = (long)p.n_items * p.n_kv_heads * head_tiles;
    const int parts = (int)max(1L, min(64L, 2L * n_sms / cells));
    const size_t bytes = STEP_WARPS * rows * (64 * VG + 2) * sizeof(float);
    static_assert(STEP_WARPS * 16 * (128 + 2) * 4 <= 100 * 1024, "two CTAs of the largest size share an SM");
    auto kernel = attention_step_kernel<KG, VG, HALVES>;
    if (bytes > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return launched(e, "attention_step");
    }
    return launched(launch_kernel(g_dependent_launch != 0, kernel, dim3(parts, p.n_kv_heads * head_tiles, p.n_items), dim3(STEP_THREADS),
                                  bytes, stream, p, head_tiles, parts),
                    "attention_step");
}

template <int HALVES>
int launch_step_of(const E4m3Attention& p, int n_sms, cudaStream_t stream) {
    if (p.dim <= 64 && p.vdim <= 64) return launch_step<1, 1, HALVES>(p, n_sms, stream);
    if (p.dim <= 64) return launch_step<1, 2, HALVES>(p, n_sms, stream);
    if (p.vdim <= 64) return launch_step<2, 1, HALVES>(p, n_sms, stream);
    return launch_step<2, 2, HALVES>(p, n_sms, stream);
}

}  // namespace

extern "C" int mllm_e4m3_store(void* q_out, long ld_q, const void* qkv, long ld, int k_off, int v_off, int heads, int kv_heads, int dim,
                               int vdim, int rot_dims, const double* inv_freq, double amplitude, const int* positions,
                               const int* token_item, const int* block_table, int max_blocks, int n_pages, int page, void* k_pages,
                               void* v_pages, float* k_scales, float* v_scales, int n, int dtype, int n_sms, void* stream) {
    if (n <= 0) return 0;
    StoreParams p = {q_out, ld_q, qkv, ld, k_off, v_off, heads, kv_heads, dim, vdim, rot_dims, inv_freq, (float)amplitude, positions,
                     token_item, block_table, max_blocks, n_pages, page, (uint8_t*)k_pages, (uint8_t*)v_pages, k_scales, v_scales, n};
    const int slots = (q_out != nullptr ? heads : 0) + (k_pages != nullptr ? 2 * kv_heads : 0);
    if (slots == 0) return 0;
    // Few rows: a CTA each, and the heads shared among as many as fill the SMs; many: sixteen, whose blocks are then one or two.
    const int G = n <= 256 ? 1 : (n <= 1024 ? 4 : 16);
    const int groups = (n + G - 1) / G, warps = STORE_THREADS / 32;
    const int share = max(1, min((slots + warps - 1) / warps, 8 * n_sms / groups));
    const size_t bytes = (size_t)(G + 15) * (rot_dims / 2) * sizeof(float2);
    const dim3 grid(groups, share);
    auto kernel = dtype == DT_BF16 ? store_kernel<bf16> : store_kernel<float>;
    return launched(launch_kernel(g_dependent_launch != 0, kernel, grid, dim3(STORE_THREADS), bytes, (cudaStream_t)stream, p, G), "e4m3_store");
}

extern "C" int mllm_e4m3_attention_plain(const E4m3Attention* p, int n_rows, int dtype, void* stream) {
    if (n_rows <= 0 || p->n_items <= 0) return 0;
    auto kernel = dtype == DT_BF16 ? attention_plain_kernel<bf16> : attention_plain_kernel<float>;
    return launched(launch_kernel(g_dependent_launch != 0, kernel, dim3(n_rows, p->n_heads), dim3(PLAIN_THREADS), 0, (cudaStream_t)stream, *p),
                    "e4m3_attention_plain");
}

extern "C" int mllm_e4m3_attention_step(const E4m3Attention* p, int n_sms, void* stream) {
    if (p->n_items <= 0) return 0;
    if (p->dim > 128 || p->vdim > 128) return fail("e4m3_attention_step: heads of more than 128 entries");
    return p->n_heads / p->n_kv_heads <= 8 ? launch_step_of<1>(*p, n_sms, (cudaStream_t)stream) : launch_step_of<2>(*p, n_sms, (cudaStream_t)stream);
}
