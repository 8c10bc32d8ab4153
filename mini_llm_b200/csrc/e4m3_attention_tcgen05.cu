// Attention of prompt portions over the 8-bit cache (e4m3.cuh) on the fifth-generation tensor cores.
//
// A CTA takes 256 consecutive tokens of an entry (a "unit": two tiles of 128 rows) and one head, and walks the keys up to the
// unit's last position in blocks of 128, or a part of them:
//   converter warps  read a block's codes, page by page, and leave them as 16-bit floats in shared memory, swizzled like a TMA tile
//                    (every code is one exactly; the scales stay outside); both tiles use them;
//   MMA warp         S = Q K^T with tcgen05.mma into tensor memory, then O += P V, P from tensor memory;
//   softmax warps    a thread a row: reads S, applies scale, cap and mask, and writes P over S as 16-bit floats.
// While one tile's softmax runs the other's products do.  Scales cost nothing an entry: a block of 16 keys has one factor for its scores, and
// its values' scale 2^t goes into the exponent, p = 2^(s + t - m + 7), with the sum of the weights getting p / 2^t; p keeps the 11 bits of a
// 16-bit float however far apart the scales lie.  Queries are scaled by a power of two to lie below 2^15.  O stays in tensor
// memory; m moves, and O is scaled down, only where a score passes m by 8 (p stays below 2^15).
//
// What bounds it is the exponential (16 a clock and SM): 2,048 clocks a unit and block, against 1,024 of the products of heads of 64.
//
// The work is laid out on the device, from the entries alone (no list is made on the host, and a replayed graph takes any
// entries): units in the order of the entries, the last of an entry first, times heads; where they are fewer than the SMs their keys
// are shared among parts, whose 32-bit results the one that arrives last adds up in order.  Every wait is bounded.
#include "common.cuh"
#include "e4m3.cuh"
#include "tcgen05.cuh"

MLLM_DEFINE_ERROR_API(mllm_e4m3_tiles)

namespace {

constexpr int TILE = 128, UNIT = 2 * TILE;
constexpr int GROUP_BYTES = TILE * 128;            // 128 rows of 64 16-bit floats
constexpr int SOFTMAX_WARPS = 8, CONVERTER_WARPS = 2, MMA_WARP = SOFTMAX_WARPS + CONVERTER_WARPS;
constexpr int THREADS = (MMA_WARP + 2) * 32;     // 384: 168 registers each
constexpr int MAX_STAGES = 4;
constexpr int MIN_PART_BLOCKS = 4;                 // blocks of 128 keys that a part has at least
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void umma_from_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_store_bits_16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
// 32 columns on their way into registers, and there (all that were asked for).
#define MLLM_32_REGISTERS(op, r) \
    op(r[0]), op(r[1]), op(r[2]), op(r[3]), op(r[4]), op(r[5]), op(r[6]), op(r[7]), op(r[8]), op(r[9]), op(r[10]), op(r[11]), op(r[12]), \
    op(r[13]), op(r[14]), op(r[15]), op(r[16]), op(r[17]), op(r[18]), op(r[19]), op(r[20]), op(r[21]), op(r[22]), op(r[23]), op(r[24]), \
    op(r[25]), op(r[26]), op(r[27]), op(r[28]), op(r[29]), op(r[30]), op(r[31])
#define MLLM_WRITTEN(x) "=r"(x)
#define MLLM_KEPT(x) "+r"(x)
__device__ __forceinline__ void tmem_ask_32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : MLLM_32_REGISTERS(MLLM_WRITTEN, r)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : MLLM_32_REGISTERS(MLLM_KEPT, r) : : "memory");
}
__device__ __forceinline__ void tmem_stores_landed() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max_of_three(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// f16 x f16 -> fp32, m x n, both operands K-major (IDESC_B_MN_MAJOR: B is not).
__device__ __forceinline__ uint32_t f16_instr_desc(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// The units of the step, as every thread can work them out from the entries.
struct Unit {
    int entry, row0, rows, pos0;                   // rows of the step, and the first one's position
    int block_lo, blocks;                          // the blocks of 128 keys that this part walks
    int part, parts, cell, index;                  // where parts of it go, and the unit's number
};

struct Schedule {
    const E4m3Attention& p;
    int units, share;                              // all units; blocks of a part, or 0: none comes in parts

    __device__ int last_block(int start, int count, int tile) const { return (start + min(count, (tile + 1) * UNIT) - 1) / TILE; }
    __device__ int first_block(int start, int tile) const {
        const int first = p.window > 0 ? start + tile * UNIT - p.window + 1 : 0;
        return first > 0 ? first / TILE : 0;
    }
    __device__ int blocks_of(int start, int count, int tile) const { return max(0, last_block(start, count, tile) - first_block(start, tile) + 1); }
    __device__ int units_of(int entry) const {
        const int count = p.item_count[entry];
        return count > 1 ? (count + UNIT - 1) / UNIT : 0;
    }
    __device__ int parts_of(int entry) const {     // of all its units
        const int n = units_of(entry);
        if (share == 0) return n;
        const int start = p.item_start[entry], count = p.item_count[entry];
        int sum = 0;
        for (int t = 0; t < n; t++) sum += max(1, (blocks_of(start, count, t) + share - 1) / share);
        return sum;
    }

    // By one whole warp, as is what is asked of it.
    __device__ explicit Schedule(const E4m3Attention& params, int n_sms) : p(params), units(0), share(0) {
        const int lane = threadIdx.x & 31;
        for (int e = lane; e < p.n_items; e += 32) units += units_of(e);
        units = __reduce_add_sync(0xffffffffu, units);
        if (units == 0 || units * p.n_heads >= n_sms) return;
        int blocks = 0;
        for (int e = lane; e < p.n_items; e += 32) {
            const int start = p.item_start[e], count = p.item_count[e];
            for (int t = units_of(e) - 1; t >= 0; t--) blocks += blocks_of(start, count, t);
        }
        blocks = __reduce_add_sync(0xffffffffu, blocks);
        share = max(MIN_PART_BLOCKS, (blocks * p.n_heads + n_sms - 1) / n_sms);
    }
    // Unit or part number `at` (over all entries); false behind the last.
    __device__ bool find(int at, Unit& u) const {
        const int lane = threadIdx.x & 31;
        int units_before = 0, before = 0;
        for (int base = 0; base < p.n_items; base += 32) {
            const int e = base + lane;
            int n = 0, parts = 0;
            if (e < p.n_items) n = units_of(e), parts = parts_of(e);
            int upto = parts, units_upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o), y = __shfl_up_sync(0xffffffffu, units_upto, o);
                if (lane >= o) upto += x, units_upto += y;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + upto > at);
            if (past != 0) {
                const int src = __ffs(past) - 1;
                u.entry = base + src;
                int left = at - before - __shfl_sync(0xffffffffu, upto - parts, src);
                int index = units_before + __shfl_sync(0xffffffffu, units_upto - n, src);
                const int start = p.item_start[u.entry], count = p.item_count[u.entry];
                int tile = units_of(u.entry) - 1;
                u.part = 0, u.parts = 1;
                if (share == 0) {
                    tile -= left, index += left;
                } else {
                    for (;; tile--, index++) {
                        u.parts = max(1, (blocks_of(start, count, tile) + share - 1) / share);
                        if (left < u.parts) break;
                        left -= u.parts;
                    }
                    u.part = left;
                }
                const int blocks = blocks_of(start, count, tile);
                const int each = (blocks + u.parts - 1) / u.parts;
                u.row0 = p.item_offset[u.entry] + tile * UNIT, u.rows = min(UNIT, count - tile * UNIT), u.pos0 = start + tile * UNIT;
                u.block_lo = first_block(start, tile) + u.part * each;
                u.blocks = max(0, min(each, blocks - u.part * each));
                u.cell = at, u.index = index;
                return true;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
            units_before += __shfl_sync(0xffffffffu, units_upto, 31);
        }
        return false;
    }
};

struct Shared {
    uint64_t unit_full[2], unit_empty[2], q_full, q_empty;
    uint64_t k_full[MAX_STAGES], k_empty[MAX_STAGES], v_full[MAX_STAGES], v_empty[MAX_STAGES];
    uint64_t s_ready[2], p_ready[2], o_ready[2], o_free[2];
    uint32_t tmem;
    int failed, ticket[2];
    Unit unit[2];                                  // entry < 0: there are no more
    int head[2];
    float q_factor[2][UNIT];
    // of the blocks of 16 keys: the keys' scale, the values' scale's exponent, and one by the values' scale
    float k_scale[MAX_STAGES][TILE / E4M3_BLOCK], v_exponent[MAX_STAGES][TILE / E4M3_BLOCK], v_inverse[MAX_STAGES][TILE / E4M3_BLOCK];
    uint4 absent[MAX_STAGES], none[MAX_STAGES];    // keys that are not there; values that are no numbers (a bit a key)
};

// (a role that gave up leaves its barriers as they are, so that the others' waits run out, or find out here)
__device__ __forceinline__ bool wait_or_fail(Shared& sh, uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    return mbar_wait(bar, parity) && !*reinterpret_cast<volatile int*>(&sh.failed);
}
__device__ __forceinline__ void give_up(Shared& sh, const E4m3Attention& p, int code) {
    if (!*reinterpret_cast<volatile int*>(&sh.failed)) {
        *reinterpret_cast<volatile int*>(&sh.failed) = 1;
        atomicExch(p.status, code);
    }
}

// A place in the ring of stages, and how often the ring has been around (its parity).  Counted, not divided: a division by a number that is not
// known beforehand costs a lone thread a hundred clocks, and several a block made the products' issue the longest chain of all.
struct Ring {
    int stage = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ Ring next(int stages) const {
        Ring r = {stage + 1, parity};
        if (r.stage == stages) r = {0, parity ^ 1};
        return r;
    }
};

// Blocks that each tile of a unit walks (the first tile's last position comes earlier).
struct Blocks {
    int n[2], most;
    __device__ explicit Blocks(const Unit& u) {
        const int last0 = u.pos0 + min(u.rows, TILE) - 1, last1 = u.pos0 + u.rows - 1;
        n[0] = last0 < 0 ? 0 : max(0, min(u.blocks, last0 / TILE - u.block_lo + 1));
        n[1] = u.rows > TILE && last1 >= 0 ? u.blocks : 0;
        most = max(n[0], n[1]);
    }
};

// A warp's next unit (the k-th it asks for); false when there are none, or a wait ran out.
__device__ __forceinline__ bool next_unit(Shared& sh, int k, Unit& u, int& head) {
    const bool ok = __all_sync(0xffffffffu, wait_or_fail(sh, &sh.unit_full[k & 1], (k >> 1) & 1));
    if (!ok) return false;
    u = sh.unit[k & 1];
    head = sh.head[k & 1];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.unit_empty[k & 1]);
    return u.entry >= 0;
}

// (two 32-bit numbers in one instruction)
__device__ __forceinline__ void fma_pair(float& x, float& y, float factor, float from) {
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(factor), "f"(from));
}
__device__ __forceinline__ void add_pair(float& x, float& y, float a, float b) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b));
}

template <bool CAP>
__global__ void __launch_bounds__(THREADS, 1) attention_tiles_kernel(const E4m3Attention p, int stages, int n_sms, int* work) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(16) Shared sh;
    dependents_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int k_groups = (p.dim + 63) / 64, v_groups = (p.vdim + 63) / 64;
    unsigned char* tiles = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    unsigned char* q_tile = tiles;                                             // [2][k_groups]
    unsigned char* k_stage = q_tile + 2 * k_groups * GROUP_BYTES;              // [stages][k_groups]
    unsigned char* v_stage = k_stage + stages * k_groups * GROUP_BYTES;        // [stages][v_groups]
    if (threadIdx.x == 0) {
        mbar_init(&sh.q_full, CONVERTER_WARPS);
        mbar_init(&sh.q_empty, 1);
        for (int s = 0; s < MAX_STAGES; s++) {
            mbar_init(&sh.k_full[s], CONVERTER_WARPS);
            mbar_init(&sh.v_full[s], CONVERTER_WARPS);
            mbar_init(&sh.k_empty[s], 1);
            mbar_init(&sh.v_empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.unit_full[i], 1);
            mbar_init(&sh.unit_empty[i], SOFTMAX_WARPS + CONVERTER_WARPS + 1);
            mbar_init(&sh.s_ready[i], 1);
            mbar_init(&sh.p_ready[i], 4);
            mbar_init(&sh.o_ready[i], 1);
            mbar_init(&sh.o_free[i], 4);
        }
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) tmem_alloc(&sh.tmem, 512);
    tcgen05_before_sync();
    __syncthreads();
    tcgen05_after_sync();
    const uint32_t tmem = sh.tmem;
    wait_for_earlier_kernels();

    Ring ring;                                      // of the next block
    if (warp < SOFTMAX_WARPS) {
        // ---- softmax: a thread a row ----
        const int tile = warp >> 2, r = threadIdx.x - tile * TILE, row = tile * TILE + r;
        const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lane_addr + TILE * tile, o_at = tmem + lane_addr + 256 + TILE * tile;
        const float cap_factor = CAP ? 2.0f * LOG2E / p.cap : 0.0f, cap_log2 = p.cap * LOG2E;
        uint32_t s_seen = 0, o_seen = 0;
        Unit u;
        int head;
        for (int k = 0; next_unit(sh, k, u, head); k++) {
            const Blocks blocks(u);
            const int n = tile == 0 ? blocks.n[0] : blocks.n[1];
            const bool has_row = row < u.rows;
            const int pos = u.pos0 + (has_row ? row : u.rows - 1);
            const int first = p.window > 0 ? pos - p.window + 1 : 0;
            const int tile_first_pos = u.pos0 + tile * TILE;
            float m = -INFINITY, l = 0.0f, q_factor = 0.0f;
            bool ok = true, sees_none = false;
            for (int j = 0; j < n; j++) {
                const int s = ring.stage, key0 = (u.block_lo + j) * TILE;
                // (the values' barrier too: what stands beside the tiles comes with it)
                ok = wait_or_fail(sh, &sh.v_full[s], ring.parity) && wait_or_fail(sh, &sh.s_ready[tile], (s_seen + j) & 1);
                ring = ring.next(stages);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tcgen05_after_sync();
                if (j == 0) q_factor = sh.q_factor[k & 1][row];
                const uint4 absent = sh.absent[s], none = sh.none[s];
                const bool needs_mask = key0 + TILE - 1 > tile_first_pos || p.window > 0 ||
                                        (absent.x | absent.y | absent.z | absent.w | none.x | none.y | none.z | none.w) != 0;
                // which of the columns c .. c + 31 this row sees
                auto seen = [&](int c) -> uint32_t {
                    const int most = pos - key0 - c, least = first - key0 - c;
                    uint32_t bits = most >= 31 ? 0xffffffffu : (most < 0 ? 0u : (2u << most) - 1u);
                    if (least > 0) bits &= least > 31 ? 0u : 0xffffffffu << least;
                    return bits & ~(c == 0 ? absent.x : c == 32 ? absent.y : c == 64 ? absent.z : absent.w);
                };
                auto mask = [&](uint32_t (&v)[32], uint32_t bits) {
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = (bits >> i) & 1 ? v[i] : 0xff800000u;
                };
                // The row is read twice, 32 columns at a time, the next ones on their way (all 128 in registers spill, and a loop body of
                // 128 columns does not stay with the instructions near the warps: 3,500 clocks a block against ...).
                // First its largest, in powers of two, with the values' scale (no factor is negative, and the cap keeps the order: the largest
                // score is the largest product's).
                float top = -INFINITY;
                uint32_t v[2][32];
                tmem_ask_32(s_at, v[0]);
                auto largest = [&](uint32_t (&x)[32], int c) {
                    if (needs_mask) {
                        const uint32_t bits = seen(c);
                        if (((c == 0 ? none.x : c == 32 ? none.y : c == 64 ? none.z : none.w) & bits) != 0) sees_none = true;
                        mask(x, bits);
                    }
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        float most[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const uint32_t* y = x + 16 * half + 8 * e;
                            most[e] = max_of_three(__uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[2]));
                            most[e] = max_of_three(most[e], __uint_as_float(y[3]), __uint_as_float(y[4]));
                            most[e] = max_of_three(most[e], __uint_as_float(y[5]), __uint_as_float(y[6]));
                            most[e] = fmaxf(most[e], __uint_as_float(y[7]));
                        }
                        const float of_all = fmaxf(most[0], most[1]);
                        const float y = of_all * (q_factor * sh.k_scale[s][c / 16 + half]), t = sh.v_exponent[s][c / 16 + half];
                        const float z = (CAP ? capped(y, cap_log2, cap_factor) : y) + t;
                        top = fmaxf(top, of_all == -INFINITY ? of_all : z);
                    }
                };
#pragma unroll 1
                for (int c = 0; c < TILE; c += 64) {
                    tmem_wait_32(v[0]);
                    tmem_ask_32(s_at + c + 32, v[1]);
                    largest(v[0], c);
                    tmem_wait_32(v[1]);
                    tmem_ask_32(s_at + ((c + 64) & (TILE - 1)), v[0]);      // (the last time: where the second reading begins)
                    largest(v[1], c + 32);
                }
                if (__any_sync(0xffffffffu, top > m + 8.0f)) {
                    const float most = fmaxf(m, top), down = m == -INFINITY ? 0.0f : exp2_fast(m - most);
                    m = most;
                    l *= down;
                    if (j > 0) {                     // (the products into O up to here are done: S of this block came behind them)
                        for (int c = 0; c < p.vdim; c += 16) {
                            float o[16];
                            tmem_load_16(o_at + c, o);
                            uint32_t w[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) w[i] = __float_as_uint(o[i] * down);
                            tmem_store_bits_16(o_at + c, w);
                        }
                    }
                }
                const float base = (m == -INFINITY ? 0.0f : m) - 7.0f;
                auto weights = [&](uint32_t (&v32)[32], int c) {
                    if (needs_mask) mask(v32, seen(c));
                    uint32_t packed[16];
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const int g = c / 16 + half;
                        const float from = sh.v_exponent[s][g] - base, factor = q_factor * sh.k_scale[s][g];
                        float sum[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float x = __uint_as_float(v32[16 * half + i]), y = __uint_as_float(v32[16 * half + i + 1]);
                            if (CAP) {
                                // (what is hidden stays hidden: its score is minus infinity, not minus the cap)
                                const float a = capped(x * factor, cap_log2, cap_factor) + from, b = capped(y * factor, cap_log2, cap_factor) + from;
                                x = x == -INFINITY ? x : a, y = y == -INFINITY ? y : b;
                            } else {
                                fma_pair(x, y, factor, from);
                            }
                            x = exp2_fast(x), y = exp2_fast(y);
                            add_pair(sum[(i >> 1) & 1][0], sum[(i >> 1) & 1][1], x, y);
                            packed[8 * half + i / 2] = half2_of(x, y);
                        }
                        add_pair(sum[0][0], sum[0][1], sum[1][0], sum[1][1]);
                        l = fmaf(sum[0][0] + sum[0][1], sh.v_inverse[s][g], l);
                    }
                    tmem_store_bits_16(s_at + c / 2, packed);      // P of columns c .. c + 31, over S, which has been read
                };
#pragma unroll 1
                for (int c = 0; c < TILE; c += 64) {
                    tmem_wait_32(v[0]);
                    tmem_ask_32(s_at + c + 32, v[1]);
                    weights(v[0], c);
                    tmem_wait_32(v[1]);
                    if (c + 64 < TILE) tmem_ask_32(s_at + c + 64, v[0]);
                    weights(v[1], c + 32);
                }
                tmem_stores_landed();
                tcgen05_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_ready[tile]);
            }
            if (ok && n > 0) {
                ok = wait_or_fail(sh, &sh.o_ready[tile], o_seen & 1);
                ok = __all_sync(0xffffffffu, ok);
                tcgen05_after_sync();
            }
            if (!ok) {
                if (lane == 0) give_up(sh, p, 34);
                break;
            }
            if (sees_none) l = __int_as_float(0x7fffffff);
            bf16* out = static_cast<bf16*>(p.out) + (u.row0 + (has_row ? row : 0)) * p.ld_out + (long)head * p.vdim;
            const int width = (p.vdim + 63) / 64 * 64;
            float* cell = p.partial + ((long)u.cell * p.n_heads + head) * UNIT * (width + 2) + row;
            if (u.parts == 1) {
                const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
                for (int c = 0; c < p.vdim; c += 16) {
                    float o[16];
                    if (n > 0) tmem_load_16(o_at + c, o);
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const __nv_bfloat162 two = n > 0 ? __floats2bfloat162_rn(o[2 * i] * inverse, o[2 * i + 1] * inverse)
                                                         : __floats2bfloat162_rn(0.0f, 0.0f);
                        w[i] = *reinterpret_cast<const uint32_t*>(&two);
                    }
                    if (has_row) {
                        *reinterpret_cast<uint4*>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
                        *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
            } else {
                // this part's sums, column by column, so that the rows of a warp lie side by side
                for (int c = 0; c < p.vdim; c += 16) {
                    float o[16];
                    if (n > 0) tmem_load_16(o_at + c, o);
#pragma unroll
                    for (int i = 0; i < 16; i++) __stcg(cell + (long)(c + i) * UNIT, n > 0 ? o[i] : 0.0f);
                }
                __stcg(cell + (long)width * UNIT, m);
                __stcg(cell + (long)(width + 1) * UNIT, l);
            }
            // O may be written again
            tcgen05_before_sync();
            __syncwarp();
            if (lane == 0 && n > 0) mbar_arrive(&sh.o_free[tile]);
            if (u.parts > 1) {
                __threadfence();
                asm volatile("bar.sync %0, 128;" ::"r"(1 + tile) : "memory");
                int* counter = p.counters + 2 * (u.index * p.n_heads + head) + tile;
                if (r == 0) sh.ticket[tile] = atomicAdd(counter, 1);
                asm volatile("bar.sync %0, 128;" ::"r"(1 + tile) : "memory");
                if (sh.ticket[tile] == u.parts - 1) {
                    __threadfence();
                    if (r == 0) *counter = 0;
                    if (has_row) {
                        const long step = (long)p.n_heads * UNIT * (width + 2);
                        const float* all = cell - u.part * step;
                        float top = -INFINITY, total = 0.0f;
                        for (int q = 0; q < u.parts; q++) top = fmaxf(top, __ldcg(all + q * step + (long)width * UNIT));
                        const float anchor = top == -INFINITY ? 0.0f : top;
                        for (int q = 0; q < u.parts; q++)
                            total += exp2_fast(__ldcg(all + q * step + (long)width * UNIT) - anchor) * __ldcg(all + q * step + (long)(width + 1) * UNIT);
                        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
                        for (int c = 0; c < p.vdim; c += 16) {
                            float o[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = 0.0f;
                            for (int q = 0; q < u.parts; q++) {
                                const float weight = exp2_fast(__ldcg(all + q * step + (long)width * UNIT) - anchor);
#pragma unroll
                                for (int i = 0; i < 16; i++) o[i] += weight * __ldcg(all + q * step + (long)(c + i) * UNIT);
                            }
                            uint32_t w[8];
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                const __nv_bfloat162 two = __floats2bfloat162_rn(o[2 * i] * inverse, o[2 * i + 1] * inverse);
                                w[i] = *reinterpret_cast<const uint32_t*>(&two);
                            }
                            *reinterpret_cast<uint4*>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
                            *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    }
                }
            }
            for (int j = n; j < blocks.most; j++) ring = ring.next(stages);
            s_seen += n;
            o_seen += n > 0 ? 1 : 0;
        }
    } else if (warp < MMA_WARP) {
        // ---- converters: a thread a key of each half of a block (and four queries) ----
        constexpr int CONVERTERS = CONVERTER_WARPS * 32, HALVES = TILE / CONVERTERS;
        const int t = threadIdx.x - SOFTMAX_WARPS * 32;
        const int k_pieces = p.dim / 16, v_pieces = p.vdim / 16;
        Unit u;
        int head;
        for (int k = 0; next_unit(sh, k, u, head); k++) {
            const int kv_head = head / (p.n_heads / p.n_kv_heads);
            const int n_blocks = Blocks(u).most, last = u.pos0 + u.rows - 1;
            const int* table = p.block_table + (long)u.entry * p.max_blocks;
            uint4 k_row[8], v_row[8];
            float k_scale = 1.0f, v_scale = 1.0f;
            bool there = false;
            // This thread's key in steps of half a block: its position, its page's place in the table and its own in the page.
            int key = u.block_lo * TILE + t, page_index = key / p.page, slot = key - page_index * p.page;
            const int key_end = min(last + 1, (u.block_lo + n_blocks) * TILE);
            auto look_up = [&](int& at_slot) -> int {        // the key's page, or -1 where it is not there; then on to the next step's
                at_slot = slot;
                int id = -1;
                if (key < key_end && page_index < p.max_blocks) id = table[page_index];
                key += CONVERTERS, slot += CONVERTERS;
                while (slot >= p.page) slot -= p.page, page_index++;
                return id < p.n_pages ? id : -1;
            };
            auto at_of = [&](int id, int at_slot) -> long { return id >= 0 ? ((long)id * p.n_kv_heads + kv_head) * p.page + at_slot : 0; };
            auto load_k = [&](int id, long at) {
                there = id >= 0;
                k_scale = v_scale = 1.0f;
                if ((t & 15) == 0 && there) k_scale = p.k_scales[at >> 4], v_scale = p.v_scales[at >> 4];
                const uint4* from = reinterpret_cast<const uint4*>(p.k_pages + at * p.dim);
#pragma unroll
                for (int i = 0; i < 8; i++) k_row[i] = (there && i < k_pieces) ? from[i] : make_uint4(0u, 0u, 0u, 0u);
            };
            auto load_v = [&](int id, long at) {
                const uint4* from = reinterpret_cast<const uint4*>(p.v_pages + at * p.vdim);
#pragma unroll
                for (int i = 0; i < 8; i++) v_row[i] = (id >= 0 && i < v_pieces) ? from[i] : make_uint4(0u, 0u, 0u, 0u);
            };
            // 16 codes to two 16-byte chunks of a row in a swizzled tile
            auto put = [&](unsigned char* stage, int row, int piece, const uint4& v) {
                uint4 a, b;
                e4m3_to_half2(v.x, a.x, a.y);
                e4m3_to_half2(v.y, a.z, a.w);
                e4m3_to_half2(v.z, b.x, b.y);
                e4m3_to_half2(v.w, b.z, b.w);
                unsigned char* at = stage + (piece >> 2) * GROUP_BYTES + row * 128;
                const int c = (piece & 3) * 2;
                *reinterpret_cast<uint4*>(at + ((c ^ (row & 7)) * 16)) = a;
                *reinterpret_cast<uint4*>(at + (((c + 1) ^ (row & 7)) * 16)) = b;
            };
            int slot_now, slot_after;
            const int id = look_up(slot_now);
            int id_after = look_up(slot_after);
            load_k(id, at_of(id, slot_now));
            load_v(id, at_of(id, slot_now));
            // the queries, once the unit before has read its own for the last time
            if (!__all_sync(0xffffffffu, wait_or_fail(sh, &sh.q_empty, (k & 1) ^ 1))) {
                if (lane == 0) give_up(sh, p, 30);
                break;
            }
            for (int row = t; row < UNIT; row += CONVERTERS) {
                const int tile = row / TILE, tile_row = row - tile * TILE;
                const bool has_row = row < u.rows;
                const uint4* from = reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q) + (u.row0 + (has_row ? row : 0)) * p.ld_q + (long)head * p.dim);
                float top = 0.0f;
                if (has_row)
#pragma unroll 4
                    for (int i = 0; i < p.dim / 8; i++) {
                        const uint4 v = from[i];
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int c = 0; c < 4; c++) top = max_of_three(top, fabsf(__uint_as_float(w[c] << 16)), fabsf(__uint_as_float(w[c] & 0xffff0000u)));
                    }
                // (zeros, and what is not finite, stay as they are)
                const int e = top > 0.0f && top < INFINITY ? max(-110, min(110, 14 - exponent_of(top))) : 0;
                const float factor = power_of_two(e);
                sh.q_factor[k & 1][row] = p.scale * power_of_two(-e) * (CAP ? 1.0f : LOG2E);
#pragma unroll 4
                for (int i = 0; i < p.dim / 8; i++) {
                    const uint4 v = has_row ? from[i] : make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    uint32_t h[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) h[c] = half2_of(__uint_as_float(w[c] << 16) * factor, __uint_as_float(w[c] & 0xffff0000u) * factor);
                    *reinterpret_cast<uint4*>(q_tile + (tile * k_groups + i / 8) * GROUP_BYTES + tile_row * 128 + (((i & 7) ^ (tile_row & 7)) * 16)) =
                        make_uint4(h[0], h[1], h[2], h[3]);
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full);
            bool ok = true;
            for (int step = 0; step < HALVES * n_blocks; step++) {
                const int half = step % HALVES, row = half * CONVERTERS + t, s = ring.stage;
                const uint32_t parity = ring.parity ^ 1;
                if (half == 0) ok = __all_sync(0xffffffffu, wait_or_fail(sh, &sh.k_empty[s], parity));
                if (!ok) break;
                const uint32_t absent = __ballot_sync(0xffffffffu, !there);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < k_pieces) put(k_stage + s * k_groups * GROUP_BYTES, row, i, k_row[i]);
                if (half == HALVES - 1) {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.k_full[s]);
                }
                // What stands beside the tiles is read until the block's P is there, which its second product waits for: behind v_empty.
                if (half == 0) ok = __all_sync(0xffffffffu, wait_or_fail(sh, &sh.v_empty[s], parity));
                if (!ok) break;
                if ((t & 15) == 0) {
                    sh.k_scale[s][row >> 4] = k_scale;
                    sh.v_exponent[s][row >> 4] = (float)exponent_of(v_scale);
                    sh.v_inverse[s][row >> 4] = 1.0f / v_scale;
                }
                const int id_now = id_after;
                const long at = at_of(id_now, slot_after);
                id_after = look_up(slot_after);
                load_k(id_now, at);
                // A value that is no number is so in its first entry; its row is left out, and the softmax puts it back in where it is seen.
                const bool none = (v_row[0].x & 0x7fu) == 0x7fu;
                const uint32_t nones = __ballot_sync(0xffffffffu, none);
                if (lane == 0) {
                    reinterpret_cast<uint32_t*>(&sh.absent[s])[row >> 5] = absent;
                    reinterpret_cast<uint32_t*>(&sh.none[s])[row >> 5] = nones;
                }
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < v_pieces) put(v_stage + s * v_groups * GROUP_BYTES, row, i, none ? make_uint4(0u, 0u, 0u, 0u) : v_row[i]);
                if (half == HALVES - 1) {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.v_full[s]);
                }
                load_v(id_now, at);
                if (half == HALVES - 1) ring = ring.next(stages);
            }
            if (!ok) {
                if (lane == 0) give_up(sh, p, 31);
                break;
            }
        }
    } else {
        if (warp == MMA_WARP) {
            // ---- products: one lane issues them ----
            const uint32_t idesc_s = f16_instr_desc(TILE, TILE), idesc_o = f16_instr_desc(TILE, p.vdim) | IDESC_B_MN_MAJOR;
            const int k_steps = p.dim / UMMA_K;
            const uint64_t q_desc = make_smem_desc(smem_u32(q_tile)), k_desc = make_smem_desc(smem_u32(k_stage));
            const uint64_t v_desc = make_smem_desc_mn(smem_u32(v_stage), GROUP_BYTES);
            uint32_t p_seen[2] = {0, 0}, o_units[2] = {0, 0};
            Unit u;
            int head;
            for (int k = 0; next_unit(sh, k, u, head); k++) {
                const Blocks blocks(u);
                bool ok = true;
                if (lane == 0) {
                    auto issue_s = [&](int tile, int s) {
                        const uint64_t a = q_desc + tile * k_groups * (GROUP_BYTES >> 4), b = k_desc + s * k_groups * (GROUP_BYTES >> 4);
                        int kk = 0;
                        for (; kk + 4 <= k_steps; kk += 4) {
                            const uint64_t group = (kk / 4) * (GROUP_BYTES >> 4);
#pragma unroll
                            for (int i = 0; i < 4; i++) umma(tmem + TILE * tile, a + group + 2 * i, b + group + 2 * i, idesc_s, kk + i > 0 ? 1u : 0u);
                        }
#pragma unroll 1
                        for (; kk < k_steps; kk++) {
                            const uint64_t at = (kk / 4) * (GROUP_BYTES >> 4) + 2 * (kk % 4);
                            umma(tmem + TILE * tile, a + at, b + at, idesc_s, kk > 0 ? 1u : 0u);
                        }
                        umma_commit(&sh.s_ready[tile]);
                    };
                    auto issue_o = [&](int tile, int s, bool begins) {
                        const uint64_t b = v_desc + s * v_groups * (GROUP_BYTES >> 4);
                        umma_from_tmem(tmem + 256 + TILE * tile, tmem + TILE * tile, b, idesc_o, begins ? 0u : 1u);
#pragma unroll
                        for (int kk = 1; kk < TILE / UMMA_K; kk++)
                            umma_from_tmem(tmem + 256 + TILE * tile, tmem + TILE * tile + kk * (UMMA_K / 2), b + kk * (2048 >> 4), idesc_o, 1u);
                    };
                    ok = wait_or_fail(sh, &sh.q_full, k & 1);
                    if (ok && blocks.most > 0) {
                        ok = wait_or_fail(sh, &sh.k_full[ring.stage], ring.parity);
                        if (ok) {
                            tcgen05_after_sync();
                            for (int tile = 0; tile < 2; tile++)
                                if (blocks.n[tile] > 0) issue_s(tile, ring.stage);
                            umma_commit(&sh.k_empty[ring.stage]);
                        }
                    }
                    for (int j = 0; ok && j < blocks.most; j++) {
                        const Ring after = ring.next(stages);
                        bool v_there = false, k_there = false;
                        for (int tile = 0; ok && tile < 2; tile++) {
                            if (j >= blocks.n[tile]) continue;
                            if (!v_there) ok = wait_or_fail(sh, &sh.v_full[ring.stage], ring.parity), v_there = true;
                            // the unit before has read its O
                            if (ok && j == 0) ok = wait_or_fail(sh, &sh.o_free[tile], (o_units[tile] & 1) ^ 1);
                            ok = ok && wait_or_fail(sh, &sh.p_ready[tile], (p_seen[tile] + j) & 1);
                            if (!ok) break;
                            tcgen05_after_sync();
                            issue_o(tile, ring.stage, j == 0);
                            if (j + 1 < blocks.n[tile]) {
                                if (!k_there) ok = wait_or_fail(sh, &sh.k_full[after.stage], after.parity), k_there = true;
                                if (!ok) break;
                                tcgen05_after_sync();
                                issue_s(tile, after.stage);
                            } else {
                                umma_commit(&sh.o_ready[tile]);
                            }
                        }
                        if (!ok) break;
                        umma_commit(&sh.v_empty[ring.stage]);
                        if (j + 1 < blocks.most) umma_commit(&sh.k_empty[after.stage]);
                        ring = after;
                    }
                    if (ok) umma_commit(&sh.q_empty);
                    else give_up(sh, p, 33);
                }
                if (!__shfl_sync(0xffffffffu, ok, 0)) break;
                for (int i = 0; i < 2; i++) p_seen[i] += blocks.n[i], o_units[i] += blocks.n[i] > 0 ? 1 : 0;
            }
        } else if (warp == MMA_WARP + 1) {
            // ---- the next unit, while the others work on this one ----
            const Schedule schedule(p, n_sms);
            for (int k = 0;; k++) {
                if (!__all_sync(0xffffffffu, wait_or_fail(sh, &sh.unit_empty[k & 1], ((k >> 1) & 1) ^ 1))) {
                    if (lane == 0) give_up(sh, p, 35);
                    break;
                }
                int at = 0;
                if (lane == 0) at = atomicAdd(work, 1);
                at = __shfl_sync(0xffffffffu, at, 0);
                Unit u;
                u.entry = -1;
                const bool more = schedule.find(at / p.n_heads, u);
                if (lane == 0) {
                    sh.unit[k & 1] = u;
                    sh.head[k & 1] = at % p.n_heads;
                    mbar_arrive(&sh.unit_full[k & 1]);
                }
                if (!more) break;
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        // the last CTA to leave puts the work counter back
        if (atomicAdd(work + 1, 1) == (int)gridDim.x - 1) work[0] = work[1] = 0;
    }
    if (warp == MMA_WARP) tmem_free(tmem, 512);
}

}  // namespace

extern "C" int mllm_e4m3_tiles_attention(const E4m3Attention* p, int n_rows, int n_sms, int* work, void* stream) {
    if (p->n_items <= 0 || n_rows <= 0) return 0;
    if (p->dim > 128 || p->vdim > 128) return fail("e4m3_attention_tiles: heads of more than 128 entries");
    const int k_groups = (p->dim + 63) / 64, v_groups = (p->vdim + 63) / 64;
    const int room = 220 * 1024 - 1024 - 2 * k_groups * GROUP_BYTES;
    const int stages = min(MAX_STAGES, room / ((k_groups + v_groups) * GROUP_BYTES));
    const size_t bytes = 1024 + (size_t)(2 * k_groups + stages * (k_groups + v_groups)) * GROUP_BYTES;
    auto kernel = p->cap > 0.0f ? attention_tiles_kernel<true> : attention_tiles_kernel<false>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return launched(e, "e4m3_attention_tiles");
    return launched(launch_kernel(g_dependent_launch != 0, kernel, dim3(n_sms), dim3(THREADS), bytes, (cudaStream_t)stream,
                                  *p, stages, n_sms, work),
                    "e4m3_attention_tiles");
}
