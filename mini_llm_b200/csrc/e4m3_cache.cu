// The 8-bit cache (e4m3.cuh): storing a step's keys and values, with the rotation of queries and keys on the way, and attention
// over it for single tokens (mma.sync tiles) and, as a plain twin for every size and type, for any row.
#include "common.cuh"
#include "e4m3.cuh"
#include "mma_tiles.cuh"

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
// table of cosines and sines serves all of them.  What bounds it is bytes, rows once in, codes and queries once out, for long
// portions (8,192 rows of 6,144 columns: 53 us, 3.5 TB/s: a lane has two pieces of 16 bytes on their way, and keys and values are walked twice), and the chain
// of positions, page and rows for single tokens (2.9 us).
constexpr int STORE_THREADS = 256, STORE_ROWS = 16;

// Eight numbers of a row, as they lie in memory.
template <typename T> struct EightOf;
template <> struct EightOf<bf16> {
    uint4 v;
    __device__ __forceinline__ void load(const bf16* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void unpack(float (&x)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
};
template <> struct EightOf<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4); }
    __device__ __forceinline__ void unpack(float (&x)[8]) const { x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w; }
};
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
    if (first >= rot_dims) return;
    if (first + 8 <= rot_dims) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const float4 two = *reinterpret_cast<const float4*>(angles + first / 2 + i);
            const float2 a = make_float2(two.x, two.y), b = make_float2(two.z, two.w);
            const float u = x[2 * i] * a.x - x[2 * i + 1] * a.y, v = x[2 * i] * a.y + x[2 * i + 1] * a.x;
            const float w = x[2 * i + 2] * b.x - x[2 * i + 3] * b.y, z = x[2 * i + 2] * b.y + x[2 * i + 3] * b.x;
            x[2 * i] = u, x[2 * i + 1] = v, x[2 * i + 2] = w, x[2 * i + 3] = z;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (first + 2 * i < rot_dims) {
            const float2 a = angles[first / 2 + i];
            const float u = x[2 * i] * a.x - x[2 * i + 1] * a.y, v = x[2 * i] * a.y + x[2 * i + 1] * a.x;
            x[2 * i] = u, x[2 * i + 1] = v;
        }
    }
}

// The larger of `most` and the squares of eight columns, as bits (what is no number, or no finite one, is the largest of all): of the lengths of pairs that
// turn, their entries times the amplitude (the square of the one or the other alone may lie beyond 32 bits where that of both does not), and of
// other entries.
__device__ __forceinline__ uint32_t largest_square(float (&x)[8], int first, int rot_dims, float amplitude, uint32_t most) {
    if (first < rot_dims && amplitude != 1.0f) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __fmul_rn(x[i], first + i < rot_dims ? amplitude : 1.0f);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = __fmul_rn(x[2 * i], x[2 * i]), b = __fmul_rn(x[2 * i + 1], x[2 * i + 1]);
        most = max(most, first + 2 * i < rot_dims ? __float_as_uint(__fadd_rn(a, b)) : max(__float_as_uint(a), __float_as_uint(b)));
    }
    return most;
}

// Sine and cosine of an eighth of a turn at most, `part` of it in 2^-32, by their Taylor series: rounded once, but for some 2^-27 of 1 before it, as from 64 bits
// (7 % of the sines and 1 % of the cosines are not the nearest 32-bit number; of a 32-bit angle 25 % and 6 % would not be).  The angle is two floats, r and a
// rest, and so are its square and 1 - r^2 / 2: what their rounding leaves joins the series' smaller terms, before the largest is added.
__device__ __forceinline__ void sine_cosine(int part, float& sine, float& cosine) {
    constexpr double UNIT = 6.283185307179586 / 4294967296.0;
    constexpr float UNIT_HIGH = (float)UNIT, UNIT_LOW = (float)(UNIT - (double)UNIT_HIGH);
    const float high = (float)part, low = (float)(part - (int)high);
    const float r = __fmul_rn(high, UNIT_HIGH);
    const float rest = __fadd_rn(__fmaf_rn(high, UNIT_HIGH, -r), __fmaf_rn(high, UNIT_LOW, __fmul_rn(low, UNIT_HIGH)));
    const float square = __fmul_rn(r, r), square_rest = __fmaf_rn(r, 2.0f * rest, __fmaf_rn(r, r, -square));
    const float half = 0.5f * square, most = __fsub_rn(1.0f, half), most_rest = __fsub_rn(__fsub_rn(1.0f, most), half);
    float a = __fmaf_rn(square, -1.0f / 39916800.0f, 1.0f / 362880.0f), b = __fmaf_rn(square, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    a = __fmaf_rn(square, a, -1.0f / 5040.0f), b = __fmaf_rn(square, b, -1.0f / 720.0f);
    a = __fmaf_rn(square, a, 1.0f / 120.0f), b = __fmaf_rn(square, b, 1.0f / 24.0f);
    a = __fmaf_rn(square, a, -1.0f / 6.0f);
    sine = __fadd_rn(r, __fmaf_rn(__fmul_rn(r, square), a, __fmul_rn(rest, most)));
    cosine = __fadd_rn(most, __fmaf_rn(__fmul_rn(square, square), b, __fmaf_rn(-0.5f, square_rest, most_rest)));
}

// A lane's pieces of eight columns of rows side by side, every 32nd, row by row: `act(row, column, numbers)` for each, the next one on its way
// (the compiler cannot know that what is stored is none of what is loaded).  One body, not unrolled: a kernel this short waits for its own
// instructions, and four pieces at a time were slower (when it was brought in: 64 rows 4.5 and 6.1 us, 8,192 rows 50 and 58).
template <typename T, typename Act>
__device__ __forceinline__ void each_piece(const T* from, long pitch, int rows, int columns, int lane, Act act) {
    const int chunks = columns / 8, step_rows = 32 / chunks, step_cols = 32 % chunks * 8;
    int row = lane / chunks, col = lane % chunks * 8;
    EightOf<T> held;
    if (row < rows) held.load(from + row * pitch + col);
#pragma unroll 1
    while (row < rows) {
        float x[8];
        held.unpack(x);
        const int row_here = row, col_here = col;
        row += step_rows, col += step_cols;
        if (col >= columns) col -= columns, row++;
        if (row < rows) held.load(from + row * pitch + col);
        act(row_here, col_here, x);
    }
}

// The least e >= -64 with square <= (448 * 2^e)^2.
__device__ __forceinline__ int scale_exponent(float square) {
    // square = m 2^x, m in [1, 2), and 448^2 = 1.53125 * 2^17
    const int bits = __float_as_int(square), x = (bits >> 23) - 127;
    const int twice = x - 17 + ((bits & 0x7fffff) > 0x440000 ? 1 : 0);          // 4^e must reach 2^twice
    return max((twice + 1) >> 1, E4M3_LEAST_EXPONENT);
}

template <typename T>
__global__ void __launch_bounds__(STORE_THREADS) store_kernel(const E4m3Store p, int G) {
    __shared__ int row_pos[STORE_ROWS + 16], row_item[STORE_ROWS + 16];        // of rows first - 1, first, ...
    __shared__ int row_page[STORE_ROWS];                                       // a leading row's page, -1: it has no place
    extern __shared__ __align__(16) float2 angles[];                           // [rows, rot_dims / 2]
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
    const uint32_t mine = p.k_pages != nullptr ? leads & ((1u << own_rows) - 1u) : 0u;
    if ((int)threadIdx.x < own_rows && ((mine >> threadIdx.x) & 1)) {
        const int pos = row_pos[threadIdx.x + 1], index = pos >= 0 ? pos / p.page : p.max_blocks;
        const int id = index < p.max_blocks ? p.block_table[(long)row_item[threadIdx.x + 1] * p.max_blocks + index] : -1;
        row_page[threadIdx.x] = id < p.n_pages ? id : -1;
    }
    int rows = own_rows;                                                       // rows whose angles are needed
    if (mine != 0) {
        const uint32_t behind = leads >> own_rows;                             // (own_rows <= 16 < 32)
        rows = min(most, own_rows + (behind != 0 ? __ffs(behind) - 1 : 31));
    }
    // Cosines and sines, a lane a pair, a warp a row: the angle in turns as a 64-bit fraction, of which whole turns fall off by themselves (what
    // rounding a frequency to 64-bit costs, 2^-53 of the angle, is all that is lost).
    const int half = p.rot_dims / 2, pitch = (half + 1) & ~1;                  // (rows on 16-byte boundaries)
    for (int i = lane; i < half; i += 32) {
        const double f = p.inv_freq[i] * 0.15915494309189535, of_turn = f - floor(f);
        const unsigned long long per_position = (unsigned long long)(of_turn * 18446744073709551616.0);
        for (int r = warp; r < rows; r += STORE_THREADS / 32) {
            const uint32_t turns = (uint32_t)((per_position * (unsigned long long)(long long)row_pos[r + 1]) >> 32);      // in 2^-32
            const uint32_t quarter = (turns + 0x20000000u) >> 30;              // the nearest
            float s, c;
            sine_cosine((int)(turns - (quarter << 30)), s, c);
            const float cosine = quarter & 1 ? -s : c, sine = quarter & 1 ? c : s, sign = quarter & 2 ? -p.amplitude : p.amplitude;
            angles[r * pitch + i] = make_float2(cosine * sign, sine * sign);
        }
    }
    __syncthreads();
    const T* qkv = behind_the_wait(static_cast<const T*>(p.qkv));
    // A warp's tasks: a head's queries of all rows, and a block's rows of a key or value head.
    const int q_tasks = p.q_out != nullptr ? p.heads : 0, slots = 2 * p.kv_heads;
    const int tasks = q_tasks + __popc(mine) * slots, stride = gridDim.y * (STORE_THREADS / 32);
    for (int task = blockIdx.y * (STORE_THREADS / 32) + warp; task < tasks; task += stride) {
        if (task < q_tasks) {
            const T* from = qkv + first * p.ld + (long)task * p.dim;
            T* to = static_cast<T*>(p.q_out) + first * p.ld_q + (long)task * p.dim;
            each_piece(from, p.ld, own_rows, p.dim, lane, [&](int row, int col, float (&x)[8]) {
                turn_eight(x, col, p.rot_dims, angles + row * pitch);
                store_eight(to + row * p.ld_q + col, x);
            });
            continue;
        }
        {
            const int lead_index = (task - q_tasks) / slots, slot = task - q_tasks - lead_index * slots;
            uint32_t todo = mine;
            for (int i = 0; i < lead_index; i++) todo &= todo - 1;
            const int r0 = __ffs(todo) - 1, page_id = row_page[r0];
            if (page_id < 0) continue;
            const bool values = slot >= p.kv_heads;
            const int head = slot - (values ? p.kv_heads : 0);
            const int size = values ? p.vdim : p.dim, rot = values ? 0 : p.rot_dims;
            const T* from = qkv + (values ? p.v_off : p.k_off) + (long)head * size + (first + r0) * p.ld;
            uint8_t* pages = values ? p.v_pages : p.k_pages;
            float* scales = values ? p.v_scales : p.k_scales;
            const uint32_t after = leads >> (r0 + 1);                          // (r0 <= 15)
            const int count = min(after != 0 ? __ffs(after) : 32, most - r0);
            const int pos = row_pos[r0 + 1], slot0 = pos % p.page, lead = pos & (E4M3_BLOCK - 1);
            const long place = (long)page_id * p.kv_heads + head;
            float* scale_at = scales + place * (p.page / E4M3_BLOCK) + slot0 / E4M3_BLOCK;
            const float held = lead > 0 ? *scale_at : 0.0f;
            uint32_t most_here = 0;
            each_piece(from, p.ld, count, size, lane, [&](int, int col, float (&x)[8]) { most_here = largest_square(x, col, rot, p.amplitude, most_here); });
            uint32_t top = __reduce_max_sync(0xffffffffu, most_here);
            uint32_t bad = 0;                                                  // rows that are not finite
            if (top >= 0x7f800000u) {
                top = 0;
                for (int r = 0; r < count; r++) {
                    most_here = 0;
                    for (int col = lane * 8; col < size; col += 256) {
                        EightOf<T> held_here;
                        float x[8];
                        held_here.load(from + r * p.ld + col);
                        held_here.unpack(x);
                        most_here = largest_square(x, col, rot, p.amplitude, most_here);
                    }
                    const uint32_t of_row = __reduce_max_sync(0xffffffffu, most_here);
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
            each_piece(from, p.ld, count, size, lane, [&](int row, int col, float (&x)[8]) {
                turn_eight(x, col, rot, angles + (r0 + row) * pitch);
                uint2 codes;
                codes.x = e4m3_pair(x[0] * inverse, x[1] * inverse) | (e4m3_pair(x[2] * inverse, x[3] * inverse) << 16);
                codes.y = e4m3_pair(x[4] * inverse, x[5] * inverse) | (e4m3_pair(x[6] * inverse, x[7] * inverse) << 16);
                if ((bad >> row) & 1) codes = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
                *reinterpret_cast<uint2*>(block + (long)(lead + row) * size + col) = codes;
            });
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
    const int first = first_seen(pos, p.window), last = last_seen(pos, p);
    for (int d = threadIdx.x; d < p.dim; d += PLAIN_THREADS)
        q[d] = to_f32(static_cast<const T*>(p.q)[row * p.ld_q + (long)head * p.dim + d]);
    float o[2] = {0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
    for (int base = first; base <= last; base += PLAIN_THREADS) {
        const int key = base + threadIdx.x, index = key / p.page;
        float s = -INFINITY;
        long at = -1;
        __syncthreads();
        if (key <= last) {
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
// The entries of one token.  What bounds them is the cache: every visible code is read once.  A unit is a token, a key/value head and up to
// eight (sixteen) of its query heads; the units stand in a row, each as long as its blocks of 16 keys and a few more for its set-up, and every
// CTA takes an equal stretch of it: requests of all lengths fill the SMs evenly, and one request alone does too.  A unit that lies in several
// stretches leaves 32-bit results of its parts, which the CTA that arrives last adds up in order.
//
// Within a CTA eight warps take a unit's blocks in turn.  A warp has its next blocks on their way into shared memory (cp.async; in
// registers one block ahead was all that fitted, 3.6 TB/s) and reads them in the layout of mma.sync m16n8k16, with the
// codes as 16-bit floats (each is one exactly) and the query heads as the eight columns:
//   S^T = K Q^T: keys g and g + 8 and columns 16 c .. 16 c + 15 of them lie with lane 4 g + c: 16 bytes each, four products; the
//     order of the columns within a product does not matter as long as Q has the same;
//   O^T = V^T P^T: keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 and columns 8 g .. 8 g + 7 of each: the pairs of keys are put together byte by byte.
// (With the heads as rows half of the products' rows are empty for up to eight heads: 632 instructions a block of 128 columns, 113 us for
// 131,072 keys of 8 heads of 128; this way 381, 58 us, and 54.5, 4.9 TB/s, since what is seldom reached is kept out of the way and no place in the
// ring is divided for.  Half of the issue slots and of the integer unit's, which converts codes, are taken then, with 16 warps an SM.)
// Q is scaled by a power of two to lie below 2^15 in 16-bit floats (11 bits: bfloat16's 8 fit; an entry 2^29 below the largest of its head
// begins to lose some, where the 32-bit sum has lost it already).  The weights: a block's value scale 2^t joins the score as t in
// the exponent, p = 2^(s + t - m + 7), and the sum of the weights gets p / 2^t, in 32 bits: no multiplication more.  m is the largest s + t (and moves
// only where a score passes it by 8, so that p stays below 2^15): a weight times its value's scale has 11 bits down to 2^-21 of the row's largest, and
// below that an error of 2^-32 of the largest, times a code of 448 at most.  (Weights as three terms of 8 bits, as for 16-bit pages, would be three
// products; a code has 4 bits.)
constexpr int STEP_WARPS = 8, STEP_THREADS = STEP_WARPS * 32, STEP_CTAS = 2;
constexpr int STEP_SET_UP = 28;                // blocks that a unit's set-up counts as (64 requests of 100 to 4,000 tokens, 8 heads of 128: 16 as many
                                               // 42.1 us, 20 39.2, 24 38.7, 28 38.3, 34 38.8)
constexpr int STEP_LEAST = 16;                 // places of a stretch, where a unit is that long
constexpr int STEP_RING_BYTES = 96 * 1024;     // of a CTA's blocks on their way

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 4 bytes to shared memory, zero where there is nothing to copy.
__device__ __forceinline__ void copy_4(void* to, const void* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(there ? 4 : 0) : "memory");
}
// An 8 x 8 tile of 16-bit numbers turned over.
__device__ __forceinline__ uint32_t turned_tile(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// All units in a row; every warp works out the same, all its lanes together.
struct StepSchedule {
    const E4m3Attention& p;
    const int units_of_entry, lane;
    long stretch, lo, hi, begin;                   // a CTA's share of the row, this CTA's, and where the unit that is next begins
    int set_up;                                    // places that a unit's set-up takes
    bool apart;                                    // every unit has CTAs of its own: it begins at a multiple of the stretch
    int entry, unit, first_block, blocks, row, pos, length;
    int base, count_of_lane, start_of_lane, row_of_lane;      // 32 entries, one a lane

    __device__ void load(int from) {
        base = from;
        const int e = from + lane;
        const bool there = e < p.n_items;
        count_of_lane = there ? p.item_count[e] : 0, start_of_lane = there ? p.item_start[e] : 0, row_of_lane = there ? p.item_offset[e] : 0;
    }
    __device__ void of_position(int position, int& lowest, int& count) const {
        lowest = first_seen(position, p.window) / E4M3_BLOCK;
        count = position >= 0 ? max(0, (last_seen(position, p) + E4M3_BLOCK) / E4M3_BLOCK - lowest) : 0;
    }
    __device__ int places(int of_blocks) const {
        if (!apart) return of_blocks + set_up;
        return (int)divided(max(of_blocks, 1) + stretch - 1, stretch) * (int)stretch;
    }
    __device__ int blocks_of_lane() const {        // -1: no unit
        if (count_of_lane != 1) return -1;
        int lowest, count;
        of_position(start_of_lane, lowest, count);
        return count;
    }
    __device__ void take(int at) {                 // the next unit is the first one of this lane's entry
        entry = base + at, unit = 0;
        row = __shfl_sync(0xffffffffu, row_of_lane, at), pos = __shfl_sync(0xffffffffu, start_of_lane, at);
        of_position(pos, first_block, blocks);
        length = places(blocks);
    }
    __device__ StepSchedule(const E4m3Attention& params, int units, int lane_) : p(params), units_of_entry(units), lane(lane_) {
        long sum = 0, entries = 0;
        int most = 0;
        for (int from = 0; from < p.n_items; from += 32) {
            load(from);
            const int n = blocks_of_lane();
            sum += __reduce_add_sync(0xffffffffu, max(n, n == 0 ? 1 : 0));
            entries += __popc(__ballot_sync(0xffffffffu, n >= 0));
            most = max(most, __reduce_max_sync(0xffffffffu, n));
        }
        sum *= units_of_entry, entries *= units_of_entry;
        // Equal stretches of the row of all units, or every unit cut by itself where that makes the longest stretch hardly longer (few units).
        const long least = min(max(most, 1), STEP_LEAST), grid = gridDim.x;
        const long together = max(divided(sum + entries * STEP_SET_UP + grid - 1, grid), least);
        stretch = entries < grid ? max(divided(sum + grid - entries - 1, grid - entries), least) : 0;
        apart = stretch > 0 && stretch <= together + STEP_SET_UP / 2;
        set_up = apart ? 0 : STEP_SET_UP;
        if (!apart) stretch = together;
        lo = blockIdx.x * stretch, hi = lo + stretch, begin = 0;
        // the unit in which the stretch begins
        for (int from = 0; from < p.n_items; from += 32) {
            if (base != from) load(from);
            const int n = blocks_of_lane(), mine = n >= 0 ? places(n) : 0;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, begin + (long)upto * units_of_entry > lo);
            if (past != 0) {
                const int at = __ffs(past) - 1;
                begin += (long)__shfl_sync(0xffffffffu, upto - mine, at) * units_of_entry;
                take(at);
                unit = (int)divided(lo - begin, length);
                begin += (long)unit * length;
                return;
            }
            begin += (long)__shfl_sync(0xffffffffu, upto, 31) * units_of_entry;
        }
        hi = lo;                                   // the row ends before
    }
    __device__ bool more() const { return begin < hi && lo < hi; }
    __device__ void next() {
        begin += length;
        if (++unit < units_of_entry || begin >= hi) return;
        uint32_t left = __ballot_sync(0xffffffffu, count_of_lane == 1) & ~((2u << (entry - base)) - 1u);
        while (left == 0 && base + 32 < p.n_items) {
            load(base + 32);
            left = __ballot_sync(0xffffffffu, count_of_lane == 1);
        }
        if (left != 0) take(__ffs(left) - 1);
        else hi = begin;                           // the row ends
    }
};

// KG, VG: groups of 64 columns of a key and a value, which they fill where EXACT; TILES: of eight query heads.
template <int KG, int VG, int TILES, bool EXACT>
__global__ void __launch_bounds__(STEP_THREADS, STEP_CTAS) attention_step_kernel(const E4m3Attention p, int head_tiles, int stages) {
    extern __shared__ __align__(128) float shared[];
    __shared__ uint4 q_parts[TILES][KG][2][32];  // the queries in the products' layout, the same for all warps
    __shared__ float q_factors[8 * TILES];       // what brings a score into powers of two
    __shared__ int ticket;
    dependents_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int dim = EXACT ? 64 * KG : p.dim, vdim = EXACT ? 64 * VG : p.vdim;
    const int group = p.n_heads / p.n_kv_heads, per_page = p.page / E4M3_BLOCK;
    constexpr float LOG2E = 1.4426950408889634f;
    constexpr int WIDTH = 64 * VG, ROWS = 8 * TILES;
    const bool has_cap = p.cap > 0.0f;
    const float cap_factor = has_cap ? 2.0f * LOG2E / p.cap : 0.0f, cap_log2 = p.cap * LOG2E;
    // a warp's ring: blocks, each behind its scales
    const int stage_bytes = 128 + E4M3_BLOCK * (dim + vdim);
    unsigned char* ring = reinterpret_cast<unsigned char*>(shared) + warp * stages * stage_bytes + 112;
    unsigned char* ring_end = ring + stages * stage_bytes;
    wait_for_earlier_kernels();
    const uint8_t* k_pages = behind_the_wait(p.k_pages);
    const uint8_t* v_pages = behind_the_wait(p.v_pages);
    StepSchedule at(p, p.n_kv_heads * head_tiles, lane);
    // A unit, or what of it lies in this stretch, and what is on its way of it while the unit before is finished.
    struct Piece {
        int row, pos, first, kv_head, head0, n_rows, lo, hi, first_cta, part, n_parts, mine;
        const int* table;
        int here, ahead;                                 // lane i: where the warp's i-th block lies (in blocks), and its i + 32nd
        uint4 q_row[KG][2];                              // the queries of tile `warp`: head g, in the order of the key's columns
    };
    // Lane i looks up 32 of the warp's blocks.
    auto look_up = [&](const Piece& u, int begins) -> int {
        const int b = begins + lane * STEP_WARPS;
        if (b >= u.hi) return -1;
        const int index = b / per_page, id = u.table[index];
        return id >= 0 && id < p.n_pages ? (id * p.n_kv_heads + u.kv_head) * per_page + b - index * per_page : -1;
    };
    auto take = [&](Piece& u) {
        u.kv_head = at.unit / head_tiles;
        const int head_tile = at.unit - u.kv_head * head_tiles;
        u.n_rows = min(ROWS, group - head_tile * ROWS), u.head0 = u.kv_head * group + head_tile * ROWS;
        u.row = at.row, u.pos = at.pos, u.first = first_seen(at.pos, p.window);
        // places of the unit in this stretch: the set-up's, then a block each
        const int from = (int)(max(at.lo, at.begin) - at.begin), to = (int)(min(at.hi, at.begin + at.length) - at.begin);
        u.lo = at.first_block + max(0, from - at.set_up), u.hi = at.first_block + min(at.blocks, max(0, to - at.set_up));
        u.first_cta = (int)divided(at.begin, at.stretch), u.n_parts = (int)divided(at.begin + at.length - 1, at.stretch) - u.first_cta + 1;
        u.part = (int)blockIdx.x - u.first_cta;
        u.table = p.block_table + (long)at.entry * p.max_blocks;
        u.mine = u.lo + warp < u.hi ? (u.hi - u.lo - warp + STEP_WARPS - 1) / STEP_WARPS : 0;
        u.here = look_up(u, u.lo + warp), u.ahead = look_up(u, u.lo + warp + 32 * STEP_WARPS);
        if (warp < TILES) {
#pragma unroll
            for (int d = 0; d < KG; d++) {
                const int col = 64 * d + 16 * c;
                const bool there = g + 8 * warp < u.n_rows && col < dim;
                const uint4* q = reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q) + u.row * p.ld_q + (long)(u.head0 + (there ? g + 8 * warp : 0)) * dim + (there ? col : 0));
                u.q_row[d][0] = there ? q[0] : make_uint4(0u, 0u, 0u, 0u);
                u.q_row[d][1] = there ? q[1] : make_uint4(0u, 0u, 0u, 0u);
            }
        }
    };
    if (!at.more()) return;
    Piece u;
    take(u);
    for (;;) {
        const int lo = u.lo, pos = u.pos, first = u.first, n_rows = u.n_rows, n_parts = u.n_parts;
        unsigned char *put = ring, *got = ring;            // where the next block goes to, and the one that is next lies
        // A block on its way: 16-byte chunks, each row's in an order in which no two lanes below read the same banks.
        auto fetch = [&](int i) {                        // the warp's i-th block, into the ring's next place
            if (i < u.mine) {
                if (__builtin_expect(i > 0 && (i & 31) == 0, 0)) u.here = u.ahead, u.ahead = look_up(u, lo + warp + (i + 32) * STEP_WARPS);
                const int place = __shfl_sync(0xffffffffu, u.here, i & 31);
                unsigned char* to = put;
                if (lane < 2) copy_4(to + 4 * lane, (lane == 0 ? p.k_scales : p.v_scales) + max(place, 0), place >= 0);     // (no scale: not there)
                if (place >= 0) {
                    const uint8_t* k = k_pages + (long)place * E4M3_BLOCK * dim;
                    const uint8_t* v = v_pages + (long)place * E4M3_BLOCK * vdim;
                    to += 16;
                    if constexpr (EXACT) {
#pragma unroll
                        for (int n = 0; n < 2 * KG; n++) {
                            const int x = lane + 32 * n, key = x / (4 * KG);
                            copy_16(to + 16 * (x ^ (KG == 2 ? (key & 1) << 2 : 0)), k + 16 * x, true);
                        }
                        to += E4M3_BLOCK * dim;
#pragma unroll
                        for (int n = 0; n < 2 * VG; n++) {
                            const int x = lane + 32 * n, key = x / (4 * VG);
                            copy_16(to + 16 * (x ^ (((key >> 1) & 3) << 1)), v + 16 * x, true);
                        }
                    } else {
                        for (int x = lane; x < dim; x += 32) copy_16(to + 16 * x, k + 16 * x, true);
                        to += E4M3_BLOCK * dim;
                        for (int x = lane; x < vdim; x += 32) copy_16(to + 16 * x, v + 16 * x, true);
                    }
                }
            }
            copies_end();
            put = put + stage_bytes == ring_end ? ring : put + stage_bytes;
        };
        for (int i = 0; i < stages - 1; i++) fetch(i);

        // the queries as 16-bit floats of a power of two's size
        if (warp < TILES) {
            const int r = g + 8 * warp;
            float x[KG][16], top = 0.0f;
#pragma unroll
            for (int d = 0; d < KG; d++) {
                const uint32_t w[8] = {u.q_row[d][0].x, u.q_row[d][0].y, u.q_row[d][0].z, u.q_row[d][0].w, u.q_row[d][1].x, u.q_row[d][1].y, u.q_row[d][1].z, u.q_row[d][1].w};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[d][2 * i] = __uint_as_float(w[i] << 16), x[d][2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                    top = fmaxf(top, fmaxf(fabsf(x[d][2 * i]), fabsf(x[d][2 * i + 1])));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = query_exponent(top);
            const float factor = power_of_two(e);
            if (c == 0) q_factors[r] = finite_factor(p.scale * power_of_two(-e) * (has_cap ? 1.0f : LOG2E));
#pragma unroll
            for (int d = 0; d < KG; d++)
#pragma unroll
                for (int s = 0; s < 2; s++)
                    q_parts[warp][d][s][lane] = make_uint4(half2_of(x[d][8 * s] * factor, x[d][8 * s + 1] * factor),
                                                           half2_of(x[d][8 * s + 2] * factor, x[d][8 * s + 3] * factor),
                                                           half2_of(x[d][8 * s + 4] * factor, x[d][8 * s + 5] * factor),
                                                           half2_of(x[d][8 * s + 6] * factor, x[d][8 * s + 7] * factor));
        }
        __syncthreads();
        // heads 2 c and 2 c + 1 of every tile are this lane's
        float q_factor[TILES][2], m[TILES][2], l[TILES][2], acc[TILES][VG][4][4];
#pragma unroll
        for (int h = 0; h < TILES; h++) {
#pragma unroll
            for (int e = 0; e < 2; e++) q_factor[h][e] = q_factors[8 * h + 2 * c + e], m[h][e] = -INFINITY, l[h][e] = 0.0f;
#pragma unroll
            for (int i = 0; i < 16 * VG; i++) acc[h][i / 16][(i / 4) & 3][i & 3] = 0.0f;
        }

        auto work = [&](const unsigned char* from, int index) {
            const float2 scales = *reinterpret_cast<const float2*>(from);
            const float k_scale = scales.x, v_scale = scales.y;
            if (v_scale == 0.0f) return;
            const unsigned char* k = from + 16;
            const unsigned char* v = k + E4M3_BLOCK * dim;
            float s[TILES][4];
#pragma unroll
            for (int h = 0; h < TILES; h++) s[h][0] = s[h][1] = s[h][2] = s[h][3] = 0.0f;
#pragma unroll
            for (int d = 0; d < KG; d++) {
                uint4 rows[2];                           // columns 64 d + 16 c .. of keys g and g + 8
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const int key = g + 8 * n, col = 64 * d + 16 * c;
                    if (EXACT) rows[n] = *reinterpret_cast<const uint4*>(k + key * dim + (col ^ (KG == 2 ? (key & 1) << 6 : 0)));
                    else rows[n] = col < dim ? *reinterpret_cast<const uint4*>(k + key * dim + col) : make_uint4(0u, 0u, 0u, 0u);
                }
                const uint32_t x[4] = {rows[0].x, rows[0].y, rows[0].z, rows[0].w}, y[4] = {rows[1].x, rows[1].y, rows[1].z, rows[1].w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t a[4];
                    e4m3_to_half2(x[i], a[0], a[2]);
                    e4m3_to_half2(y[i], a[1], a[3]);
#pragma unroll
                    for (int h = 0; h < TILES; h++) {
                        const uint4 q = q_parts[h][d][i >> 1][lane];
                        mma_f16(s[h], a, (i & 1) ? q.z : q.x, (i & 1) ? q.w : q.y);
                    }
                }
            }
            const float t = (float)exponent_of(v_scale), over = 1.0f / v_scale;
            const int key0 = index * E4M3_BLOCK;
            const bool partial = key0 + E4M3_BLOCK - 1 > pos || key0 < first;
            const float after = has_cap ? 0.0f : t;
            // scores of key g, heads 2 c and 2 c + 1, then of key g + 8
            float top[TILES][2];
            bool moves = false;
#pragma unroll
            for (int h = 0; h < TILES; h++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float factor = q_factor[h][e] * k_scale;
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        s[h][2 * n + e] = fmaf(s[h][2 * n + e], factor, after);
                    }
                    if (__builtin_expect(has_cap, 0)) {
                        s[h][e] = capped(s[h][e], cap_log2, cap_factor) + t, s[h][2 + e] = capped(s[h][2 + e], cap_log2, cap_factor) + t;
                    }
                    if (__builtin_expect(partial, 0)) {
                        if (key0 + g > pos || key0 + g < first) s[h][e] = -INFINITY;
                        if (key0 + g + 8 > pos || key0 + g + 8 < first) s[h][2 + e] = -INFINITY;
                    }
                    top[h][e] = fmaxf(s[h][e], s[h][2 + e]);
                    moves = moves || top[h][e] > m[h][e] + 8.0f;
                }
            if (__builtin_expect(__any_sync(0xffffffffu, moves), 0)) {
#pragma unroll
                for (int h = 0; h < TILES; h++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float most = top[h][e];
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                        most = fmaxf(m[h][e], most);
                        const float down = m[h][e] == -INFINITY ? 0.0f : exp2_fast(m[h][e] - most);
                        m[h][e] = most;
                        l[h][e] *= down;
#pragma unroll
                        for (int d = 0; d < VG; d++)
#pragma unroll
                            for (int n = 0; n < 4; n++) acc[h][d][n][e] *= down, acc[h][d][n][2 + e] *= down;
                    }
            }
            uint32_t weights[TILES][2];
#pragma unroll
            for (int h = 0; h < TILES; h++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float base = (m[h][e] == -INFINITY ? 0.0f : m[h][e]) - 7.0f;
                    s[h][e] = exp2_fast(s[h][e] - base);
                    s[h][2 + e] = exp2_fast(s[h][2 + e] - base);
                    l[h][e] = fmaf(s[h][e] + s[h][2 + e], over, l[h][e]);
                }
                weights[h][0] = turned_tile(half2_of(s[h][0], s[h][1]));
                weights[h][1] = turned_tile(half2_of(s[h][2], s[h][3]));
            }
#pragma unroll
            for (int d = 0; d < VG; d++) {
                uint2 rows[4];                           // columns 64 d + 8 g .. of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const int key = 2 * c + (n & 1) + 8 * (n >> 1), col = 64 * d + 8 * g;
                    if (EXACT) rows[n] = *reinterpret_cast<const uint2*>(v + ((key * vdim + col) ^ (((key >> 1) & 3) << 5)));
                    else rows[n] = col < vdim ? *reinterpret_cast<const uint2*>(v + key * vdim + col) : make_uint2(0u, 0u);
                }
                // (a masked key's value may be no number, and its weight of zero would not keep it out)
                if (__builtin_expect(partial, 0)) {
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const int key = key0 + 2 * c + (n & 1) + 8 * (n >> 1);
                        if (key > pos || key < first) rows[n] = make_uint2(0u, 0u);
                    }
                }
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    // columns 2 n and 2 n + 1 of the eight: keys a and b of the one, then of the other
                    const uint32_t order = (n & 1) ? 0x7362 : 0x5140;
                    uint32_t a[4];
                    e4m3_to_half2(__byte_perm(n >> 1 ? rows[0].y : rows[0].x, n >> 1 ? rows[1].y : rows[1].x, order), a[0], a[1]);
                    e4m3_to_half2(__byte_perm(n >> 1 ? rows[2].y : rows[2].x, n >> 1 ? rows[3].y : rows[3].x, order), a[2], a[3]);
#pragma unroll
                    for (int h = 0; h < TILES; h++) mma_f16(acc[h][d][n], a, weights[h][0], weights[h][1]);
                }
            }
        };
        for (int i = 0; i < u.mine; i++) {
            // block i has landed (as many groups behind it are on their way as the ring has places but two), and all lanes have left block i - 1
            if (stages == 4) copies_landed<2>();
            else if (stages == 3) copies_landed<1>();
            else copies_landed<4>();
            __syncwarp();
            fetch(i + stages - 1);
            work(got, lo + warp + i * STEP_WARPS);
            got = got + stage_bytes == ring_end ? ring : got + stage_bytes;
        }
        copies_landed<0>();
        __syncthreads();                                 // the ring's memory is the results' now

        // the warps' results: rows of sums, then the maxima and the sums of the weights
        float* of_m = shared + STEP_WARPS * n_rows * WIDTH;
        float* of_l = of_m + STEP_WARPS * n_rows;
#pragma unroll
        for (int h = 0; h < TILES; h++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], o);
                const int r = 8 * h + 2 * c + e;
                if (r < n_rows) {
                    if (g == 0) of_m[warp * n_rows + r] = m[h][e], of_l[warp * n_rows + r] = l[h][e];
                    float* sums = shared + (warp * n_rows + r) * WIDTH + 8 * g;
#pragma unroll
                    for (int d = 0; d < VG; d++)
#pragma unroll
                        for (int n = 0; n < 4; n += 2)
                            *reinterpret_cast<float4*>(sums + 64 * d + 2 * n) =
                                make_float4(acc[h][d][n][e], acc[h][d][n][2 + e], acc[h][d][n + 1][e], acc[h][d][n + 1][2 + e]);
                }
            }
        __syncthreads();
        // the next unit's pages and queries come while this one's results are put together
        const int row = u.row, head0 = u.head0, first_cta = u.first_cta, part = u.part;
        at.next();
        const bool more = at.more();
        if (more) take(u);
        bf16* out = static_cast<bf16*>(p.out) + row * p.ld_out + (long)head0 * vdim;
        // A part that begins a unit is its CTA's last and has the second of the CTA's two places; any other is its first.
        constexpr int PART = ROWS * (WIDTH + 2);
        auto cell = [&](int q) { return p.partial + (long)(2 * (first_cta + q) + (q == 0 ? 1 : 0)) * PART; };
        for (int i = threadIdx.x; i < n_rows * WIDTH; i += STEP_THREADS) {
            const int r = i / WIDTH, col = i - r * WIDTH;
            float top = -INFINITY, sum = 0.0f, weight_sum = 0.0f;
#pragma unroll
            for (int w = 0; w < STEP_WARPS; w++) top = fmaxf(top, of_m[w * n_rows + r]);
            const float anchor = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < STEP_WARPS; w++) {
                const float weight = exp2_fast(of_m[w * n_rows + r] - anchor);
                sum += weight * shared[(w * n_rows + r) * WIDTH + col];
                weight_sum += weight * of_l[w * n_rows + r];
            }
            if (n_parts == 1) {
                if (col < vdim) out[r * vdim + col] = __float2bfloat16_rn(weight_sum == 0.0f ? 0.0f : sum / weight_sum);
            } else {
                float* here = cell(part);
                __stcg(here + i, sum);
                if (col == 0) __stcg(reinterpret_cast<float2*>(here + ROWS * WIDTH + 2 * r), make_float2(top, weight_sum));
            }
        }
        if (n_parts > 1) {
            __threadfence();
            __syncthreads();
            int* counter = p.counters + first_cta;
            if (threadIdx.x == 0) ticket = atomicAdd(counter, 1);
            __syncthreads();
            if (ticket == n_parts - 1) {
                __threadfence();
                // The last to arrive adds the parts up, in their order: two columns a thread, eight parts on their way at a time.
                constexpr int AT_ONCE = 8;
                for (int i = 2 * threadIdx.x; i < n_rows * WIDTH; i += 2 * STEP_THREADS) {
                    const int r = i / WIDTH, col = i - r * WIDTH;
                    float top = -INFINITY, weight_sum = 0.0f;
                    float2 sum = make_float2(0.0f, 0.0f);
                    for (int q0 = 0; q0 < n_parts; q0 += AT_ONCE) {
                        float2 of_part[AT_ONCE], state[AT_ONCE];
#pragma unroll
                        for (int n = 0; n < AT_ONCE; n++) {
                            of_part[n] = make_float2(0.0f, 0.0f), state[n] = make_float2(-INFINITY, 0.0f);
                            if (q0 + n < n_parts) {
                                const float* theirs = cell(q0 + n);
                                of_part[n] = __ldcg(reinterpret_cast<const float2*>(theirs + i));
                                state[n] = __ldcg(reinterpret_cast<const float2*>(theirs + ROWS * WIDTH + 2 * r));
                            }
                        }
                        float most = top;
#pragma unroll
                        for (int n = 0; n < AT_ONCE; n++) most = fmaxf(most, state[n].x);
                        const float anchor = most == -INFINITY ? 0.0f : most, down = exp2_fast(top - anchor);
                        sum.x *= down, sum.y *= down, weight_sum *= down, top = most;
#pragma unroll
                        for (int n = 0; n < AT_ONCE; n++) {
                            const float weight = exp2_fast(state[n].x - anchor);
                            sum.x += weight * of_part[n].x, sum.y += weight * of_part[n].y, weight_sum += weight * state[n].y;
                        }
                    }
                    const float inverse = weight_sum == 0.0f ? 0.0f : 1.0f / weight_sum;
                    if (col < vdim) *reinterpret_cast<__nv_bfloat162*>(out + r * vdim + col) = __floats2bfloat162_rn(sum.x * inverse, sum.y * inverse);
                }
                if (threadIdx.x == 0) *counter = 0;
            }
        }
        if (!more) break;
        __syncthreads();                                 // (shared memory is the next unit's)
    }
}

template <int KG, int VG, int TILES, bool EXACT>
int launch_step(const E4m3Attention& p, int n_sms, cudaStream_t stream) {
    const int group = p.n_heads / p.n_kv_heads, rows = min(group, 8 * TILES);
    const int head_tiles = (group + 8 * TILES - 1) / (8 * TILES);
    const int stage_bytes = 128 + E4M3_BLOCK * (p.dim + p.vdim), of_all = STEP_WARPS * stage_bytes;
    const int stages = of_all * 6 <= STEP_RING_BYTES ? 6 : of_all * 4 <= STEP_RING_BYTES ? 4 : 3;
    const size_t bytes = max((size_t)stages * of_all, STEP_WARPS * rows * (64 * VG + 2) * sizeof(float));
    constexpr size_t MOST = 3 * STEP_WARPS * (128 + E4M3_BLOCK * 256);
    static_assert(MOST <= 104 * 1024 && STEP_RING_BYTES <= MOST && STEP_WARPS * 16 * (128 + 2) * 4 <= MOST, "two CTAs of the largest size share an SM");
    auto kernel = attention_step_kernel<KG, VG, TILES, EXACT>;
    static std::atomic<bool> raised[64];
    const cudaError_t e = raise_shared_limit(kernel, MOST, raised);
    if (e != cudaSuccess) return launched(e, "e4m3_attention_step");
    // as many CTAs as the SMs hold, or as the longest row that the tables allow is cut into
    const long units = (long)p.n_items * p.n_kv_heads * head_tiles, most = (long)p.max_blocks * (p.page / E4M3_BLOCK);
    const int grid = (int)max(1L, min((long)STEP_CTAS * n_sms, units * ((most + STEP_LEAST - 1) / STEP_LEAST + 1)));
    return launched(launch_kernel(g_dependent_launch != 0, kernel, dim3(grid), dim3(STEP_THREADS), bytes, stream, p, head_tiles, stages),
                    "e4m3_attention_step");
}

template <int TILES>
int launch_step_of(const E4m3Attention& p, int n_sms, cudaStream_t stream) {
    if (p.dim == 64 && p.vdim == 64) return launch_step<1, 1, TILES, true>(p, n_sms, stream);
    if (p.dim == 128 && p.vdim == 128) return launch_step<2, 2, TILES, true>(p, n_sms, stream);
    if (p.dim <= 64 && p.vdim <= 64) return launch_step<1, 1, TILES, false>(p, n_sms, stream);
    return launch_step<2, 2, TILES, false>(p, n_sms, stream);
}

}  // namespace

extern "C" int mllm_e4m3_store(const E4m3Store* operands, int dtype, int n_sms, void* stream) {
    const E4m3Store& p = *operands;
    const int n = p.n, rot_dims = p.rot_dims;
    if (n <= 0) return 0;
    const int slots = (p.q_out != nullptr ? p.heads : 0) + (p.k_pages != nullptr ? 2 * p.kv_heads : 0);
    if (slots == 0) return 0;
    // Rows a CTA, and the heads shared among as many CTAs as fill the SMs.  Single tokens, of which each begins a block, want few rows a CTA,
    // long portions many, whose angles are then made once (when it was brought in, rows a CTA 4, 8, 16: a portion of 1,500 with shorter ones and 40 single tokens
    // 10.5, 11.3, 15.9 us; 8,192 rows of 40 turned heads of 128 64.9, 55.8, 53.8).
    const int G = n <= 256 ? 1 : (n <= 4096 ? 4 : 16);
    const int groups = (n + G - 1) / G, warps = STORE_THREADS / 32;
    const int share = max(1, min((slots + warps - 1) / warps, 16 * n_sms / groups));
    const size_t bytes = (size_t)(G + 15) * ((rot_dims / 2 + 1) & ~1) * sizeof(float2);
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
