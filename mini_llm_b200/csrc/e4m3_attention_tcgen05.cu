// Attention of prompt portions over the 8-bit cache (e4m3.cuh) on the fifth-generation tensor cores.
//
// A unit is 256 consecutive tokens of an entry (two tiles of 128 rows) and one head; a CTA walks the keys up to the unit's last
// position in blocks of 128:
//   converter warps  read a block's codes, page by page, and leave them as 16-bit floats in shared memory, swizzled like a TMA tile
//                    (every code is one exactly; the scales stay outside); both tiles use them;
//   MMA warp         S = Q K^T with tcgen05.mma into tensor memory, then O += P V, P from tensor memory;
//   softmax warps    two threads a row, each with 64 of a block's columns: read S, apply scale, cap and mask, write P as 16-bit floats; and, since they have
//                    nothing else to do at a unit's start, its queries.
// While one tile's softmax runs the other's products do.  Scales cost nothing an entry: a block of 16 keys has one factor for its scores, and
// its values' scale 2^t goes into the exponent, p = 2^(s + t - m + 7), with the sum of the weights getting p / 2^t in 32 bits; p, a weight times its value's
// scale, is a 16-bit float: 11 bits down to 2^-21 of the row's largest, below an error of 2^-32 of the largest, times a code of 448 at most.  Queries are scaled by a power of two to lie below 2^15.  O stays in tensor
// memory; m moves, and O is scaled down, only where a score passes m by 8 (p stays below 2^15).
//
// A unit and block takes the exponential's unit 2,048 clocks (16 a clock and SM), the tensor cores 1,024 with heads of 64 and 2,048 with 128, and reads
// next to nothing from memory.  It takes 4,250 clocks with heads of 64 (a prompt of 16,000 tokens, 12 heads: 738 us, half of the exponential's rate) and
// 5,250 with 128 (2,000 tokens behind 14,000, 32 heads: 577 us, 0.87 PFLOP/s): what lies between is the chain of a tile's turn, S, its largest, the
// tile's meeting, the weights, P, which the other tile's turn fills in part, and the instruction fetch of four roles at once.  Without exponentials,
// largest and conversion the chain alone still took 667 us of 766 in an earlier state.
//
// The work is laid out on the device, from the entries alone (no list is made on the host, and a replayed graph takes any
// entries): the units, each as long as its blocks and one more, stand in a row, and every CTA takes an equal stretch of it.  A unit that
// lies in several stretches leaves 32-bit results of its parts, which the CTA that arrives last adds up in order.  Where there are few units each is cut
// by itself instead, so that no CTA begins two.  Every wait is bounded.
#include "common.cuh"
#include "e4m3.cuh"
#include "tcgen05.cuh"

MLLM_DEFINE_ERROR_API(mllm_e4m3_tiles)

namespace {

constexpr int TILE = 128, UNIT = 2 * TILE;
constexpr int GROUP_BYTES = TILE * 128;            // 128 rows of 64 16-bit floats
constexpr int SOFTMAX_WARPS = 16, CONVERTER_WARPS = 4, MMA_WARP = SOFTMAX_WARPS + CONVERTER_WARPS;
constexpr int THREADS = (MMA_WARP + 4) * 32;       // (the last two warps only make the fourth warp of their group up)
// Registers a thread: all start with the same, and the last four warps, which need few, give up what the softmax warps take.  The shares never add up
// to more than the block was launched with (`registers_suffice`).  When it was brought in: 790 us for 16,000 tokens of 12 heads of 64 without, 766 with it.
constexpr int SOFTMAX_REGISTERS = 88, IDLE_REGISTERS = 48;
constexpr bool registers_suffice(int at_launch) {
    return THREADS / 32 * at_launch >= SOFTMAX_WARPS * SOFTMAX_REGISTERS + CONVERTER_WARPS * at_launch + 4 * IDLE_REGISTERS && at_launch >= IDLE_REGISTERS &&
           at_launch <= SOFTMAX_REGISTERS;
}
constexpr int MAX_STAGES = 4;
constexpr int MIN_STRETCH = 5;                     // of a CTA, where no unit is longer: its blocks and one more
constexpr int MIN_STRETCH_APART = 4;               // the same where every unit is cut by itself, in blocks (prompts of 300, 400, 500, 700 and 1,000 tokens, 12 heads
                                                   // of 64: 2 14.5, 16.5, 17.4, 18.5, 21.3 us; 3 12.2, 19.6, 20.3, 20.5, 21.3; 4 12.2, 16.0, 16.6, 21.6,
                                                   // 22.0; 5 12.2, 16.0, 16.6, 24.4, 24.8; of 300, 400 and 500, 32 heads of 128: 2 20.3, 26.7, 28.4; 3 15.6,
                                                   // 26.7, 28.5; 4 15.6, 20.6, 21.3)
constexpr float LOG2E = 1.4426950408889634f;

// What one thread of the MMA warp does while all of its lanes run: a warp that does not branch apart keeps descriptors where the
// instruction wants them (issued by a lane that is alone in a branch, each product took 70 to 120 clocks of moves).
__device__ __forceinline__ uint32_t elected_lane() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is;
}
__device__ __forceinline__ void umma_by(uint32_t elected, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(elected)
        : "memory");
}
__device__ __forceinline__ void umma_from_tmem_by(uint32_t elected, uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(elected)
        : "memory");
}
__device__ __forceinline__ void umma_commit_by(uint32_t elected, uint64_t* bar) {
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(elected)
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

// A piece of work: a unit, or the part of it that lies in this CTA's stretch.
struct Unit {
    int entry, row0, rows, pos0;                   // rows of the step, and the first one's position
    int block_lo, blocks;                          // the blocks of 128 keys
    int part, parts, first_cta;                    // of the unit, and the CTA with its first part
    int head;
};

// All units in a row, by one whole warp.
struct Schedule {
    const E4m3Attention& p;
    long total, stretch, lo, hi;                   // the row's length, a CTA's share, this CTA's
    long begin;                                    // of the unit that is next
    int entry, tile, head, blocks, length, start, count, offset;
    int base, count_of_lane, start_of_lane, offset_of_lane;          // 32 entries, one a lane
    int set_up;                                    // places that a unit's set-up takes
    bool apart;                                    // every unit has CTAs of its own: it begins at a multiple of the stretch

    __device__ void load(int from, int lane) {
        base = from;
        const int e = from + lane;
        const bool there = e < p.n_items;
        count_of_lane = there ? p.item_count[e] : 0, start_of_lane = there ? p.item_start[e] : 0, offset_of_lane = there ? p.item_offset[e] : 0;
    }
    __device__ int first_block(int s, int t) const {
        return first_seen(s + t * UNIT, p.window) / TILE;
    }
    __device__ int blocks_of(int s, int c, int t) const {
        const int last = last_seen(s - 1 + min(c, (t + 1) * UNIT), p);
        return last < 0 ? 0 : max(0, last / TILE - first_block(s, t) + 1);
    }
    __device__ int places(int of_blocks) const {
        return apart ? (max(of_blocks, 1) + (int)stretch - 1) / (int)stretch * (int)stretch : of_blocks + set_up;
    }
    __device__ static int tiles_of(int c) { return (c + UNIT - 1) / UNIT; }

    __device__ Schedule(const E4m3Attention& params, int lane) : p(params), total(0), entry(-1) {
        int sum = 0, none = 0, most = 0, units = 0;         // blocks of this lane's units, those without any, the longest; all units
        for (int from = 0; from < p.n_items; from += 32) {
            load(from, lane);
            for (uint32_t bits = __ballot_sync(0xffffffffu, count_of_lane > 1); bits != 0; bits &= bits - 1) {
                const int c = __shfl_sync(0xffffffffu, count_of_lane, __ffs(bits) - 1), s = __shfl_sync(0xffffffffu, start_of_lane, __ffs(bits) - 1);
                for (int t = lane; t < tiles_of(c); t += 32) {
                    const int n = blocks_of(s, c, t);
                    sum += n, none += n == 0 ? 1 : 0, most = max(most, n);
                }
                units += tiles_of(c);
            }
        }
        // Equal stretches of the row of all units, or, where there are fewer units than CTAs, every unit cut by itself, if that makes the longest
        // stretch no longer.
        const long all = (long)__reduce_add_sync(0xffffffffu, sum) * p.n_heads, of_units = (long)units * p.n_heads, grid = gridDim.x;
        const long cut = all + (long)__reduce_add_sync(0xffffffffu, none) * p.n_heads;
        most = __reduce_max_sync(0xffffffffu, most);
        const long together = max(divided(all + of_units + grid - 1, grid), (long)min(most + 1, MIN_STRETCH));
        const long by_itself = of_units < grid ? max(divided(cut + grid - of_units - 1, grid - of_units), (long)min(max(most, 1), MIN_STRETCH_APART)) : 0;
        apart = by_itself > 0 && by_itself <= together;
        set_up = apart ? 0 : 1;
        stretch = apart ? by_itself : together;
        total = apart ? grid * stretch : all + of_units;         // (no longer than that, where the units stand apart)
        lo = blockIdx.x * stretch, hi = min(total, lo + stretch);
        if (lo >= hi) return;
        // the unit in which the stretch begins
        begin = 0;
        for (int from = 0; from < p.n_items; from += 32) {
            if (base != from) load(from, lane);
            for (uint32_t bits = __ballot_sync(0xffffffffu, count_of_lane > 1); bits != 0; bits &= bits - 1) {
                const int src = __ffs(bits) - 1;
                const int c = __shfl_sync(0xffffffffu, count_of_lane, src), s = __shfl_sync(0xffffffffu, start_of_lane, src), n = tiles_of(c);
                for (int first = 0; first < n; first += 32) {
                    const int t = n - 1 - first - lane;
                    const int of_lane = t >= 0 ? blocks_of(s, c, t) : 0, mine = t >= 0 ? places(of_lane) : 0;
                    int upto = mine;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int x = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += x;
                    }
                    const uint32_t past = __ballot_sync(0xffffffffu, begin + (long)upto * p.n_heads > lo);
                    if (past != 0) {
                        const int at = __ffs(past) - 1;
                        length = __shfl_sync(0xffffffffu, mine, at), blocks = __shfl_sync(0xffffffffu, of_lane, at);
                        begin += (long)__shfl_sync(0xffffffffu, upto - mine, at) * p.n_heads;
                        head = (int)divided(lo - begin, length);
                        begin += (long)head * length;
                        entry = base + src, tile = n - 1 - first - at, start = s, count = c;
                        offset = __shfl_sync(0xffffffffu, offset_of_lane, src);
                        return;
                    }
                    begin += (long)__shfl_sync(0xffffffffu, upto, 31) * p.n_heads;
                }
            }
        }
        hi = lo;                                   // the row ends before
    }
    __device__ bool next(Unit& u) {
        if (lo >= hi || begin >= hi) return false;
        const long end = begin + length;
        const int from = (int)(max(lo, begin) - begin), to = (int)(min(hi, end) - begin);      // place 0 is the unit's set-up
        u.entry = entry, u.head = head;
        u.row0 = offset + tile * UNIT, u.rows = min(UNIT, count - tile * UNIT), u.pos0 = start + tile * UNIT;
        u.block_lo = first_block(start, tile) + max(0, from - set_up);
        u.blocks = min(blocks, max(0, to - set_up)) - max(0, from - set_up);
        u.first_cta = (int)divided(begin, stretch);
        u.parts = (int)divided(end - 1, stretch) - u.first_cta + 1;
        u.part = (int)blockIdx.x - u.first_cta;
        begin = end;
        if (++head == p.n_heads && begin < hi) {
            head = 0;
            if (--tile < 0) {
                do entry++; while (p.item_count[entry] <= 1);          // (the row goes on, so there is one)
                start = p.item_start[entry], count = p.item_count[entry], offset = p.item_offset[entry];
                tile = tiles_of(count) - 1;
            }
            blocks = blocks_of(start, count, tile), length = places(blocks);
        }
        return true;
    }
};

struct Shared {
    uint64_t unit_full[2], unit_empty[2], q_full[2];
    uint64_t k_full[MAX_STAGES], k_empty[MAX_STAGES], v_full[MAX_STAGES], v_empty[MAX_STAGES];
    uint64_t s_ready[2], s_read[2], p_ready[2], o_added[2], o_free[2];
    uint32_t tmem;
    int failed, ticket[2];
    Unit unit[2];                                  // entry < 0: there are no more
    float q_factor[UNIT];
    float of_half[2][2][TILE];                     // what the two threads of a row tell one another
    // of the blocks of 16 keys: the keys' scale, the values' scale's exponent, and one by the values' scale
    float k_scale[MAX_STAGES][TILE / E4M3_BLOCK], v_exponent[MAX_STAGES][TILE / E4M3_BLOCK], v_inverse[MAX_STAGES][TILE / E4M3_BLOCK];
    alignas(8) uint32_t absent[MAX_STAGES][4];     // keys that are not there, and whose values are no numbers (a bit a key; read two words at a time)
    alignas(8) uint32_t none[MAX_STAGES][4];
    // (last: 12 bytes more ahead of the units move what is read in the loops, 616 us for 573 of 2,000 tokens at the end of 16,000)
    uint32_t wait_limit;                           // of every wait, in ns
    alignas(8) uint64_t all_done;
};

// Codes of the roles that give up.
constexpr int CONVERTERS_GAVE_UP = 31, PRODUCTS_GAVE_UP = 33, SOFTMAX_GAVE_UP = 34, SCHEDULE_GAVE_UP = 35;

// (a role that gave up leaves its barriers as they are; the others find out here)
// By a whole warp, with one answer for all of its lanes: what follows does not branch apart, and the compiler knows it.  Code that is seldom reached
// is kept out of the way here and in the softmax: 24 warps in four roles share the instruction caches, and what they fetch past, they wait for
// (when it was brought in: a prompt of 16,000 766 us and 2,000 tokens at its end of 32 heads of 128 612 us with all of it in line, 704 and 574 this way).
__device__ __forceinline__ bool wait_or_fail(Shared& sh, uint64_t* bar, uint32_t parity) {
    if (__builtin_expect(__any_sync(0xffffffffu, mbar_try_wait(bar, parity)), 1)) return true;
    const uint32_t start = (uint32_t)now_ns();       // (32 bits of it: looks lie microseconds apart, and the limit is below 2^31)
    do {
#pragma unroll 1
        for (int i = 0; i < 256; i++)
            if (__any_sync(0xffffffffu, mbar_try_wait(bar, parity))) return !__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&sh.failed));
    } while (!__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&sh.failed) || (uint32_t)now_ns() - start > sh.wait_limit));
    return false;
}
__device__ __forceinline__ void give_up(Shared& sh, const E4m3Attention& p, int code) {
    if (!*reinterpret_cast<volatile int*>(&sh.failed)) {
        *reinterpret_cast<volatile int*>(&sh.failed) = 1;
        atomicExch(p.status, code);
    }
}

// A place in the ring of stages, and how often the ring has been around (its parity).  Counted, not divided: a division by a number that is not
// known beforehand costs a lone thread a hundred clocks, and several a block made the products' issue the longest chain of all.
// A wait by parity is exact only where the phase before the one that is meant is known to be over.  A role that walks every block knows it from its
// own waits.  A softmax tile passes over the blocks of a unit in which it has no rows (or fewer) without waiting, so that it waits for a ring's
// barrier only behind s_ready, whose phases it counts itself: S of a block is made when all converter warps have put the block's keys, which
// each does after the values of the block before, and so after all earlier blocks of the stage.
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
        const int last0 = u.pos0 - 1 + min(u.rows, TILE), last1 = u.pos0 - 1 + u.rows;
        n[0] = last0 < 0 ? 0 : max(0, min(u.blocks, last0 / TILE - u.block_lo + 1));
        n[1] = u.rows > TILE && last1 >= 0 ? u.blocks : 0;
        most = max(n[0], n[1]);
    }
};

// A warp's next unit (the k-th it asks for); false when there are none, or (`ok`) a wait ran out.
__device__ __forceinline__ bool next_unit(Shared& sh, int k, Unit& u, bool& ok) {
    ok = wait_or_fail(sh, &sh.unit_full[k & 1], (k >> 1) & 1);
    if (!ok) return false;
    u = sh.unit[k & 1];
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

__device__ __forceinline__ void mul_pair(float& x, float& y, float a, float b) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b));
}
__device__ __forceinline__ void fma_pairs(float& x, float& y, float a, float b, float from) {
    asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %4};\n\t"
        "fma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b), "f"(from));
}

// A factor of scores is never zero, which no hidden score's minus infinity would outlast: queries or a scale that small make scores of nothing either way.
__device__ __forceinline__ float never_zero(float factor) { return fmaxf(factor, 0x1p-126f); }

// 32 products (two blocks of 16 keys) to capped scores.  Up to a quarter of the cap, where scores mostly lie, by the series of tanh u / u in u^2 to its
// third power (the next term is 2^-23.5 of the cap there): otherwise the exponential's unit, which the weights need, has two more operations a score (a
// portion of 1,024 behind 1,345 and two short prompts, 12 heads of 64: 48.0 us, and 41.3).  One score beyond sends a warp's 32 rows the other way: a prompt of
// 8,000 takes 208 us without a cap, 311 with scores below a quarter of it and 390 with scores far beyond.
__device__ __forceinline__ void cap_scores(uint32_t (&v)[32], float q_factor, const float* k_scale, float cap_log2, float cap_factor, float by_cap) {
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        float x = __uint_as_float(v[i]), y = __uint_as_float(v[i + 1]);
        const float factor = never_zero(q_factor * k_scale[i / 16]);
        mul_pair(x, y, factor, factor);
        far = max_of_three(far, fabsf(x), fabsf(y));
        v[i] = __float_as_uint(x), v[i + 1] = __float_as_uint(y);
    }
    if (__builtin_expect(__any_sync(0xffffffffu, far > 0.25f * cap_log2), 0)) {
#pragma unroll
        for (int i = 0; i < 32; i++) {
            // (what is hidden stays hidden: its score is minus infinity, not minus the cap)
            const float x = __uint_as_float(v[i]);
            v[i] = __float_as_uint(x == -INFINITY ? x : capped(x, cap_log2, cap_factor));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const float x = __uint_as_float(v[i]), y = __uint_as_float(v[i + 1]);
        float a = x, b = y;
        mul_pair(a, b, by_cap, by_cap);
        mul_pair(a, b, a, b);
        float p = a, q = b;
        fma_pair(p, q, -17.0f / 315.0f, 2.0f / 15.0f);
        fma_pairs(p, q, a, b, -1.0f / 3.0f);
        fma_pairs(p, q, a, b, 1.0f);
        mul_pair(p, q, x, y);
        v[i] = __float_as_uint(p), v[i + 1] = __float_as_uint(q);
    }
}

// The 256 threads of a tile meet; whether any of them says yes.  (Where a wait ran out for some of them only, they leave together all the same,
// from a meeting in which one said so: one that left alone would keep the others waiting here for good.)
__device__ __forceinline__ bool any_of_tile(int tile, bool yes) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any)
                 : "r"(1 + tile), "r"(yes ? 1u : 0u)
                 : "memory");
    return any != 0;
}
__device__ __forceinline__ void tile_meets(int tile) { asm volatile("barrier.cta.sync %0, 256;" ::"r"(1 + tile) : "memory"); }

__device__ __forceinline__ void store_sixteen(bf16* to, const float (&o)[16], float factor) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(o[2 * i] * factor, o[2 * i + 1] * factor);
        w[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(to + 8) = make_uint4(w[4], w[5], w[6], w[7]);
}

// 16 rows of a unit's queries into shared memory, by a warp, eight or sixteen lanes a row: as 16-bit floats of a power of two's size, and what
// brings a row's scores into powers of two.
template <int GROUPS>
__device__ __forceinline__ void put_queries(const E4m3Attention& p, const Unit& u, unsigned char* to, float* factors, int first_row, int lane) {
    constexpr int LANES = 8 * GROUPS, ROWS = 32 / LANES, AT_ONCE = 4, OF_WARP = UNIT / SOFTMAX_WARPS;
    const int chunk = lane % LANES, row0 = first_row + lane / LANES;
    const bf16* from = static_cast<const bf16*>(p.q) + (long)u.row0 * p.ld_q + (long)u.head * p.dim + 8 * chunk;
#pragma unroll 1
    for (int base = 0; base < OF_WARP; base += AT_ONCE * ROWS) {
        uint4 v[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) {
            const int row = row0 + base + i * ROWS;
            v[i] = row < u.rows && 8 * chunk < p.dim ? *reinterpret_cast<const uint4*>(from + row * p.ld_q) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) {
            const int row = row0 + base + i * ROWS;
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            float top = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; c++) top = max_of_three(top, fabsf(__uint_as_float(w[c] << 16)), fabsf(__uint_as_float(w[c] & 0xffff0000u)));
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = query_exponent(top);
            const float factor = power_of_two(e);
            if (chunk == 0) factors[row] = finite_factor(p.scale * power_of_two(-e) * LOG2E);
            uint32_t h[4];
#pragma unroll
            for (int c = 0; c < 4; c++) h[c] = half2_of(__uint_as_float(w[c] << 16) * factor, __uint_as_float(w[c] & 0xffff0000u) * factor);
            *reinterpret_cast<uint4*>(to + ((row / TILE) * GROUPS + chunk / 8) * GROUP_BYTES + (row % TILE) * 128 + (((chunk ^ row) & 7) * 16)) =
                make_uint4(h[0], h[1], h[2], h[3]);
        }
    }
    fence_async_smem();
}

// GROUPS: groups of 64 columns that a key and a value take in shared memory.
// Tensor memory: S of the tiles from columns 0 and 128 on.  With one group O lies from 256 and 320 on, and P, which two 16-bit floats a column
// make half as wide, from 384 and 448 on, so that S of the next block need not wait for the product with P; with two, O from 256 and
// 384 on, and P over S, each half of a row's columns over the first half of its own.
template <bool CAP, int GROUPS>
__global__ void __launch_bounds__(THREADS, 1) attention_tiles_kernel(const E4m3Attention p, int stages) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(16) Shared sh;
    dependents_may_start();
    constexpr bool P_APART = GROUPS == 1;
    constexpr int O_AT = 2 * TILE, O_STEP = 64 * GROUPS, P_AT = P_APART ? 384 : 0, P_STEP = P_APART ? 64 : TILE, P_HALF = P_APART ? 32 : 64;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* tiles = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    unsigned char* q_tile = tiles;                                             // [2][GROUPS]
    unsigned char* k_stage = q_tile + 2 * GROUPS * GROUP_BYTES;                // [stages][GROUPS]
    unsigned char* v_stage = k_stage + stages * GROUPS * GROUP_BYTES;          // [stages][GROUPS]
    if (threadIdx.x == 0) {
        for (int s = 0; s < MAX_STAGES; s++) {
            mbar_init(&sh.k_full[s], CONVERTER_WARPS);
            mbar_init(&sh.v_full[s], CONVERTER_WARPS);
            mbar_init(&sh.k_empty[s], 1);
            mbar_init(&sh.v_empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.q_full[i], SOFTMAX_WARPS / 2);
            mbar_init(&sh.unit_full[i], 1);
            mbar_init(&sh.unit_empty[i], SOFTMAX_WARPS + CONVERTER_WARPS + 1);
            mbar_init(&sh.s_ready[i], 1);
            mbar_init(&sh.s_read[i], SOFTMAX_WARPS / 2);
            mbar_init(&sh.p_ready[i], SOFTMAX_WARPS / 2);
            mbar_init(&sh.o_added[i], 1);
            mbar_init(&sh.o_free[i], SOFTMAX_WARPS / 2);
        }
        mbar_init(&sh.all_done, 1);
        sh.failed = 0;
        sh.wait_limit = p.wait_limit_ns > 0 ? p.wait_limit_ns : (uint32_t)WAIT_LIMIT_NS;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) tmem_alloc(&sh.tmem, 512);
    tcgen05_before_sync();
    __syncthreads();
    tcgen05_after_sync();
    const uint32_t tmem = sh.tmem;
    wait_for_earlier_kernels();

    Ring ring;                                      // of the next block
    Unit u;
    if (warp < SOFTMAX_WARPS) {
        // ---- softmax: two threads a row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGISTERS));
        const int tile = warp >> 3, half = (warp >> 2) & 1, r = (warp & 3) * 32 + lane, row = tile * TILE + r;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_at = lanes + TILE * tile + 64 * half, o_at = lanes + O_AT + O_STEP * tile, p_at = lanes + P_AT + P_STEP * tile + P_HALF * half;
        // (scores are in powers of two from the first on, and so is the cap)
        const float cap_log2 = p.cap * LOG2E, cap_factor = CAP ? 2.0f / p.cap : 0.0f, by_cap = CAP ? 1.0f / cap_log2 : 0.0f;
        uint32_t seen_blocks = 0;                    // of this tile, over all units
        bool ok = true;
        for (int k = 0; p.role_away != SOFTMAX_GAVE_UP; k++) {
            const bool more = next_unit(sh, k, u, ok);
            if (any_of_tile(tile, !ok)) ok = false;
            if (!ok || !more) break;
            const Blocks blocks(u);
            const int n = tile == 0 ? blocks.n[0] : blocks.n[1];
            // The tile's queries: the last unit's have been read for the last time (its last S was there), and there is nothing else to do before there are
            // some.  (When it was brought in: the converter warps took 11,000 clocks for them with heads of 128, ahead of a unit's first keys: a prompt of 100 tokens 9.8 us
            // for 8.1, 500 behind 3,000 67 for 61.  Where units are many and long they had them ready ahead: 16,000 tokens 707 us for 732.)
            if (n > 0) {
                put_queries<GROUPS>(p, u, q_tile, sh.q_factor, warp * (UNIT / SOFTMAX_WARPS), lane);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.q_full[tile]);
            }
            const bool has_row = row < u.rows;
            const int pos = u.pos0 + (has_row ? row : u.rows - 1);
            const int first = first_seen(pos, p.window);
            const int unseen = first_seen(u.pos0 - 1 + min(u.rows, (tile + 1) * TILE), p.window) - 1;      // keys up to here some row of the tile does not see
            float m = -INFINITY, l = 0.0f, q_factor = 0.0f;
            bool sees_none = false;
            for (int j = 0; j < n; j++, seen_blocks++) {
                const int s = ring.stage, key0 = (u.block_lo + j) * TILE + 64 * half;
                // The values' barrier too: what stands beside the tiles comes with it.  Behind S, not ahead of it: a tile that has passed over blocks does not
                // know how far the converters are, and takes a phase two older for the one it means; that S is there shows the older one over.
                ok = wait_or_fail(sh, &sh.s_ready[tile], seen_blocks & 1) && wait_or_fail(sh, &sh.v_full[s], ring.parity);
                ring = ring.next(stages);
                tcgen05_after_sync();
                if (j == 0) q_factor = sh.q_factor[row];
                const uint2 absent = *reinterpret_cast<const uint2*>(&sh.absent[s][2 * half]), none = *reinterpret_cast<const uint2*>(&sh.none[s][2 * half]);
                const bool needs_mask = key0 + 63 > u.pos0 + tile * TILE || key0 <= unseen || (absent.x | absent.y | none.x | none.y) != 0;
                // which of the columns c .. c + 31 this row sees
                auto seen = [&](int c) -> uint32_t {
                    const int most = pos - key0 - c, least = first - key0 - c;
                    uint32_t bits = most >= 31 ? 0xffffffffu : (most < 0 ? 0u : (2u << most) - 1u);
                    if (least > 0) bits &= least > 31 ? 0u : 0xffffffffu << least;
                    return bits & ~(c == 0 ? absent.x : absent.y);
                };
                auto mask = [&](uint32_t (&v)[32], uint32_t bits) {
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = (bits >> i) & 1 ? v[i] : 0xff800000u;
                };
                // The row is read twice, 32 columns at a time (a loop body of all of them does not stay with the instructions near the warps: 4 %
                // slower; 16 at a time are 3 % slower too, and so is the next chunk asked for before this one is worked on, 17 %).
                // First its largest, in powers of two, with the values' scale (no factor is negative, and the cap keeps the order: the largest
                // score is the largest product's).
                float top = -INFINITY;
                uint32_t v[32];
#pragma unroll 1
                for (int c = 0; ok && c < 64; c += 32) {
                    tmem_ask_32(s_at + c, v);
                    tmem_wait_32(v);
                    if (__builtin_expect(needs_mask, 0)) {
                        const uint32_t bits = seen(c);
                        if (((c == 0 ? none.x : none.y) & bits) != 0) sees_none = true;
                        mask(v, bits);
                        tmem_store_bits_16(s_at + c, v), tmem_store_bits_16(s_at + c + 16, v + 16);      // (the second reading has no mask)
                        tmem_stores_landed();
                    }
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        float most[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const uint32_t* y = v + 16 * g + 8 * e;
                            most[e] = max_of_three(__uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[2]));
                            most[e] = max_of_three(most[e], __uint_as_float(y[3]), __uint_as_float(y[4]));
                            most[e] = max_of_three(most[e], __uint_as_float(y[5]), __uint_as_float(y[6]));
                            most[e] = fmaxf(most[e], __uint_as_float(y[7]));
                        }
                        const int group = 4 * half + c / 16 + g;
                        const float of_all = fmaxf(most[0], most[1]);
                        const float y = of_all * (q_factor * sh.k_scale[s][group]);
                        const float z = (CAP ? capped(y, cap_log2, cap_factor) : y) + sh.v_exponent[s][group];
                        top = fmaxf(top, of_all == -INFINITY ? of_all : z);
                    }
                }
                // the product before has been added to O, and has read its P
                if (j > 0) ok = ok && wait_or_fail(sh, &sh.o_added[tile], (seen_blocks - 1) & 1);
                if (any_of_tile(tile, top > m + 8.0f || !ok)) {
                    sh.of_half[tile][half][r] = top;
                    if (any_of_tile(tile, !ok)) {
                        ok = false;
                        break;
                    }
                    const float most = fmaxf(m, fmaxf(top, sh.of_half[tile][half ^ 1][r])), down = m == -INFINITY ? 0.0f : exp2_fast(m - most);
                    m = most;
                    l *= down;
                    if (j > 0) {
                        tcgen05_after_sync();
                        for (int c = 16 * half; c < p.vdim; c += 32) {       // (the two threads take turns with 16 columns)
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
#pragma unroll 1
                for (int c = 0; c < 64; c += 32) {
                    tmem_ask_32(s_at + c, v);
                    tmem_wait_32(v);
                    if (P_APART && c == 32) {
                        // S may be written again
                        tcgen05_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.s_read[tile]);
                    }
                    uint32_t packed[16];
                    if (CAP) cap_scores(v, q_factor, &sh.k_scale[s][4 * half + c / 16], cap_log2, cap_factor, by_cap);
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        const int group = 4 * half + c / 16 + g;
                        const float from = sh.v_exponent[s][group] - base, factor = CAP ? 1.0f : never_zero(q_factor * sh.k_scale[s][group]);
                        float sum[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float x = __uint_as_float(v[16 * g + i]), y = __uint_as_float(v[16 * g + i + 1]);
                            if (CAP) add_pair(x, y, from, from);
                            else fma_pair(x, y, factor, from);
                            x = exp2_fast(x), y = exp2_fast(y);
                            add_pair(sum[(i >> 1) & 1][0], sum[(i >> 1) & 1][1], x, y);
                            packed[8 * g + i / 2] = half2_of(x, y);
                        }
                        add_pair(sum[0][0], sum[0][1], sum[1][0], sum[1][1]);
                        l = fmaf(sum[0][0] + sum[0][1], sh.v_inverse[s][group], l);
                    }
                    tmem_store_bits_16(p_at + c / 2, packed);
                }
                tmem_stores_landed();
                tcgen05_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_ready[tile]);
            }
            if (!ok) break;                          // (all 256 threads)
            if (n > 0) ok = wait_or_fail(sh, &sh.o_added[tile], (seen_blocks - 1) & 1);
            for (int j = n; j < blocks.most; j++) ring = ring.next(stages);
            if (sees_none) l = __int_as_float(0x7fffffff);
            sh.of_half[tile][half][r] = l;
            if (any_of_tile(tile, !ok)) {
                ok = false;
                break;
            }
            tcgen05_after_sync();
            l += sh.of_half[tile][half ^ 1][r];
            bf16* out = static_cast<bf16*>(p.out) + (u.row0 + (has_row ? row : 0)) * p.ld_out + (long)u.head * p.vdim;
            // Parts leave their sums column by column, so that the rows of a warp lie side by side.  A part that begins a unit is its CTA's last and has
            // the second of the CTA's two places; any other is its first.
            const int width = p.vdim <= 64 ? 64 : 128, rows_of_cell = width + 2;
            auto cell = [&](int part) { return p.partial + (long)(2 * (u.first_cta + part) + (part == 0 ? 1 : 0)) * UNIT * rows_of_cell + row; };
            float* mine = cell(u.part);
            const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
            for (int c = 16 * half; c < p.vdim; c += 32) {
                float o[16];
                if (n > 0) {
                    tmem_load_16(o_at + c, o);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = 0.0f;
                }
                if (u.parts == 1) {
                    if (has_row) store_sixteen(out + c, o, inverse);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) __stcg(mine + (c + i) * UNIT, o[i]);
                }
            }
            // O may be written again
            tcgen05_before_sync();
            __syncwarp();
            if (lane == 0 && n > 0) mbar_arrive(&sh.o_free[tile]);
            if (u.parts > 1) {
                if (half == 0) __stcg(mine + width * UNIT, m), __stcg(mine + (width + 1) * UNIT, l);
                __threadfence();
                tile_meets(tile);
                int* counter = p.counters + 2 * u.first_cta + tile;
                if (half == 0 && r == 0) sh.ticket[tile] = atomicAdd(counter, 1);
                tile_meets(tile);
                if (sh.ticket[tile] == u.parts - 1) {
                    __threadfence();
                    if (half == 0 && r == 0) *counter = 0;
                    if (has_row) {
                        float top = -INFINITY, total = 0.0f;
                        for (int q = 0; q < u.parts; q++) top = fmaxf(top, __ldcg(cell(q) + width * UNIT));
                        const float anchor = top == -INFINITY ? 0.0f : top;
                        for (int q = 0; q < u.parts; q++)
                            total += exp2_fast(__ldcg(cell(q) + width * UNIT) - anchor) * __ldcg(cell(q) + (width + 1) * UNIT);
                        for (int c = 16 * half; c < p.vdim; c += 32) {
                            float o[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = 0.0f;
                            for (int q = 0; q < u.parts; q++) {
                                const float* theirs = cell(q);
                                const float weight = exp2_fast(__ldcg(theirs + width * UNIT) - anchor);
#pragma unroll
                                for (int i = 0; i < 16; i++) o[i] += weight * __ldcg(theirs + (c + i) * UNIT);
                            }
                            store_sixteen(out + c, o, total == 0.0f ? 0.0f : 1.0f / total);
                        }
                    }
                }
            }
        }
        if (!ok && lane == 0) give_up(sh, p, SOFTMAX_GAVE_UP);
    } else if (warp < MMA_WARP && p.role_away == CONVERTERS_GAVE_UP) {
        // (a test's switch; within the loop below it makes registers spill)
    } else if (warp < MMA_WARP) {
        // ---- converters: a thread a key ----
        const int t = threadIdx.x - SOFTMAX_WARPS * 32;
        bool ok = true;
        for (int k = 0; next_unit(sh, k, u, ok); k++) {
            const int kv_head = u.head / (p.n_heads / p.n_kv_heads);
            const int n_blocks = Blocks(u).most;
            const int* table = p.block_table + (long)u.entry * p.max_blocks;
            // This thread's key, block after block: its position, its page's place in the table and its own in the page.
            int key = u.block_lo * TILE + t, page_index = key / p.page, slot = key - page_index * p.page;
            const int key_last = min(u.pos0 - 1 + u.rows, (u.block_lo + n_blocks) * TILE - 1);
            auto look_up = [&]() -> int {                    // the key's page, or -1 where it is not there
                const int id = key <= key_last && page_index < p.max_blocks ? table[page_index] : -1;
                return id < p.n_pages ? id : -1;
            };
            auto row_of = [&](int id) -> long { return id >= 0 ? ((long)id * p.n_kv_heads + kv_head) * p.page + slot : -1; };
            auto go_on = [&]() {
                key += TILE, slot += TILE;
                while (slot >= p.page) slot -= p.page, page_index++;
            };
            // 64 columns of a key or a value
            auto fetch = [&](uint4 (&to)[4], const uint8_t* pages, int size, int group, long at) {
                const uint4* from = reinterpret_cast<const uint4*>(pages + max(at, 0L) * size + 64 * group);
#pragma unroll
                for (int i = 0; i < 4; i++) to[i] = at >= 0 && 64 * group + 16 * i < size ? from[i] : make_uint4(0u, 0u, 0u, 0u);
            };
            // 16 codes are two 16-byte chunks of a row in a swizzled tile
            auto put = [&](unsigned char* group, const uint4 (&v)[4]) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint4 a, b;
                    e4m3_to_half2(v[i].x, a.x, a.y);
                    e4m3_to_half2(v[i].y, a.z, a.w);
                    e4m3_to_half2(v[i].z, b.x, b.y);
                    e4m3_to_half2(v[i].w, b.z, b.w);
                    *reinterpret_cast<uint4*>(group + t * 128 + (((2 * i) ^ (t & 7)) * 16)) = a;
                    *reinterpret_cast<uint4*>(group + t * 128 + (((2 * i + 1) ^ (t & 7)) * 16)) = b;
                }
            };
            // A value that is no number is so from its first entry on.  Its row is left out of the tile, where a weight of zero would not keep it
            // out of other rows, and the softmax puts it back in where it is seen.
            auto put_value = [&](unsigned char* group, uint4 (&v)[4], bool none) {
                if (none) v[0] = v[1] = v[2] = v[3] = make_uint4(0u, 0u, 0u, 0u);
                put(group, v);
            };
            const int id_first = look_up();
            long at = row_of(id_first);
            go_on();
            float k_scale = 1.0f, v_scale = 1.0f;
            auto scales = [&]() {
                k_scale = v_scale = 1.0f;
                if ((t & 15) == 0 && at >= 0) k_scale = p.k_scales[at >> 4], v_scale = p.v_scales[at >> 4];
            };
            uint4 buffer[2][4];                              // on their way: the next 128 columns, keys' before values'
            fetch(buffer[0], p.k_pages, p.dim, 0, at);
            if (GROUPS == 2) fetch(buffer[1], p.k_pages, p.dim, 1, at);
            else fetch(buffer[1], p.v_pages, p.vdim, 0, at);
            scales();
            for (int j = 0; j < n_blocks; j++) {
                const int s = ring.stage;
                const uint32_t parity = ring.parity ^ 1;
                const int id_next = look_up();
                ok = wait_or_fail(sh, &sh.k_empty[s], parity);
                if (!ok) break;
                unsigned char* k_tile = k_stage + s * GROUPS * GROUP_BYTES;
                unsigned char* v_tile = v_stage + s * GROUPS * GROUP_BYTES;
                const uint32_t absent = __ballot_sync(0xffffffffu, at < 0);
                put(k_tile, buffer[0]);
                const long at_next = row_of(id_next);
                if (GROUPS == 2) {
                    fetch(buffer[0], p.v_pages, p.vdim, 0, at);
                    put(k_tile + GROUP_BYTES, buffer[1]);
                    fetch(buffer[1], p.v_pages, p.vdim, 1, at);
                } else {
                    fetch(buffer[0], p.k_pages, p.dim, 0, at_next);
                }
                go_on();
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.k_full[s]);
                // What stands beside the tiles is read until the block's P is there, which its second product waits for: behind v_empty.
                ok = wait_or_fail(sh, &sh.v_empty[s], parity);
                if (!ok) break;
                if ((t & 15) == 0) {
                    sh.k_scale[s][t >> 4] = k_scale;
                    sh.v_exponent[s][t >> 4] = (float)exponent_of(v_scale);
                    sh.v_inverse[s][t >> 4] = 1.0f / v_scale;
                }
                at = at_next;
                scales();
                const bool none = (buffer[GROUPS == 2 ? 0 : 1][0].x & 0x7fu) == 0x7fu;
                if (GROUPS == 2) {
                    put_value(v_tile, buffer[0], none);
                    fetch(buffer[0], p.k_pages, p.dim, 0, at);
                    put_value(v_tile + GROUP_BYTES, buffer[1], none);
                    fetch(buffer[1], p.k_pages, p.dim, 1, at);
                } else {
                    put_value(v_tile, buffer[1], none);
                    fetch(buffer[1], p.v_pages, p.vdim, 0, at);
                }
                const uint32_t nones = __ballot_sync(0xffffffffu, none);
                if (lane == 0) sh.absent[s][warp - SOFTMAX_WARPS] = absent, sh.none[s][warp - SOFTMAX_WARPS] = nones;
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.v_full[s]);
                ring = ring.next(stages);
            }
            if (!ok) break;
        }
        if (!ok && lane == 0) give_up(sh, p, CONVERTERS_GAVE_UP);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(IDLE_REGISTERS));
        if (warp == MMA_WARP) {
            // ---- products ----
            const uint32_t elected = elected_lane();
            const uint32_t idesc_s = f16_instr_desc(TILE, TILE), idesc_o = f16_instr_desc(TILE, p.vdim) | IDESC_B_MN_MAJOR;
            const uint64_t q_desc = make_smem_desc(smem_u32(q_tile)), k_desc = make_smem_desc(smem_u32(k_stage));
            const uint64_t v_desc = make_smem_desc_mn(smem_u32(v_stage), GROUP_BYTES);
            const uint32_t tmem0 = __shfl_sync(0xffffffffu, tmem, 0);
            uint32_t seen_blocks[2] = {0, 0}, seen_units[2] = {0, 0};
                auto issue_s = [&](int tile, int s) {
                const uint64_t a = q_desc + tile * GROUPS * (GROUP_BYTES >> 4), b = k_desc + s * GROUPS * (GROUP_BYTES >> 4);
#pragma unroll
                for (int kk = 0; kk < 4 * GROUPS; kk++) {          // (entries behind `dim` are zeros on both sides)
                    const uint64_t at = (kk / 4) * (GROUP_BYTES >> 4) + 2 * (kk % 4);
                    umma_by(elected, tmem0 + TILE * tile, a + at, b + at, idesc_s, kk > 0 ? 1u : 0u);
                }
                umma_commit_by(elected, &sh.s_ready[tile]);
            };
            auto issue_o = [&](int tile, int s, bool begins) {
                const uint64_t b = v_desc + s * GROUPS * (GROUP_BYTES >> 4);
                const uint32_t a = tmem0 + P_AT + P_STEP * tile, d = tmem0 + O_AT + O_STEP * tile;
                umma_from_tmem_by(elected, d, a, b, idesc_o, begins ? 0u : 1u);
#pragma unroll
                for (int kk = 1; kk < TILE / UMMA_K; kk++)
                    umma_from_tmem_by(elected, d, a + (kk / 4) * P_HALF + (kk % 4) * (UMMA_K / 2), b + kk * (2048 >> 4), idesc_o, 1u);
                umma_commit_by(elected, &sh.o_added[tile]);
            };
            bool ok = true;
            for (int k = 0; p.role_away != PRODUCTS_GAVE_UP && next_unit(sh, k, u, ok); k++) {
                const Blocks of_unit(u);
                // (the same for all lanes, and the compiler knows it)
                const int n0 = __shfl_sync(0xffffffffu, of_unit.n[0], 0), n1 = __shfl_sync(0xffffffffu, of_unit.n[1], 0), most = max(n0, n1);
                if (most > 0) {
                    ok = wait_or_fail(sh, &sh.k_full[ring.stage], ring.parity);
#pragma unroll
                    for (int tile = 0; tile < 2; tile++) {
                        if ((tile == 0 ? n0 : n1) == 0) continue;
                        ok = ok && wait_or_fail(sh, &sh.q_full[tile], seen_units[tile] & 1);
                        if (!ok) break;
                        tcgen05_after_sync();
                        issue_s(tile, ring.stage);
                    }
                    if (!ok) break;
                    umma_commit_by(elected, &sh.k_empty[ring.stage]);
                }
                for (int j = 0; j < most; j++) {
                    const Ring after = ring.next(stages);
                    ok = wait_or_fail(sh, &sh.v_full[ring.stage], ring.parity);
                    if (j + 1 < most) ok = ok && wait_or_fail(sh, &sh.k_full[after.stage], after.parity);
#pragma unroll
                    for (int tile = 0; tile < 2; tile++) {
                        const int n = tile == 0 ? n0 : n1;
                        if (j >= n) continue;
                        const uint32_t parity = (seen_blocks[tile] + j) & 1;
                        if (P_APART && j + 1 < n) {
                            ok = ok && wait_or_fail(sh, &sh.s_read[tile], parity);
                            if (!ok) break;
                            tcgen05_after_sync();
                            issue_s(tile, after.stage);
                        }
                        // the unit before has read its O
                        if (j == 0) ok = ok && wait_or_fail(sh, &sh.o_free[tile], (seen_units[tile] & 1) ^ 1);
                        ok = ok && wait_or_fail(sh, &sh.p_ready[tile], parity);
                        if (!ok) break;
                        tcgen05_after_sync();
                        issue_o(tile, ring.stage, j == 0);
                        if (!P_APART && j + 1 < n) issue_s(tile, after.stage);
                    }
                    if (!ok) break;
                    umma_commit_by(elected, &sh.v_empty[ring.stage]);
                    if (j + 1 < most) umma_commit_by(elected, &sh.k_empty[after.stage]);
                    ring = after;
                }
                if (!ok) break;
                seen_blocks[0] += n0, seen_blocks[1] += n1;
                seen_units[0] += n0 > 0 ? 1 : 0, seen_units[1] += n1 > 0 ? 1 : 0;
            }
            if (!ok && lane == 0) give_up(sh, p, PRODUCTS_GAVE_UP);
            // No product is on its way any more, whether all went well or a role gave up, when the memory that they read and write is given back.
            umma_commit_by(elected, &sh.all_done);
            mbar_wait(&sh.all_done, 0);
        } else if (warp == MMA_WARP + 1) {
            // ---- the next unit, while the others work on this one ----
            Schedule schedule(p, lane);
            for (int k = 0; p.role_away != SCHEDULE_GAVE_UP; k++) {
                if (!wait_or_fail(sh, &sh.unit_empty[k & 1], ((k >> 1) & 1) ^ 1)) {
                    if (lane == 0) give_up(sh, p, SCHEDULE_GAVE_UP);
                    break;
                }
                u.entry = -1;
                const bool more = schedule.next(u);
                if (lane == 0) {
                    sh.unit[k & 1] = u;
                    mbar_arrive(&sh.unit_full[k & 1]);
                }
                if (!more) break;
            }
        }
    }
    tcgen05_before_sync();
    __syncthreads();
    tcgen05_after_sync();
    if (warp == MMA_WARP) tmem_free(tmem, 512);
}

}  // namespace

extern "C" int mllm_e4m3_tiles_attention(const E4m3Attention* p, int n_rows, int n_sms, void* stream) {
    if (p->n_items <= 0 || n_rows <= 0) return 0;
    if (p->dim > 128 || p->vdim > 128) return fail("e4m3_attention_tiles: heads of more than 128 entries");
    const int groups = p->dim <= 64 && p->vdim <= 64 ? 1 : 2, stages = groups == 1 ? 4 : 2;
    const size_t bytes = 1024 + (size_t)(2 + 2 * stages) * groups * GROUP_BYTES;
    const int which = (p->cap > 0.0f ? 2 : 0) + groups - 1;
    static std::atomic<bool> raised[4][64];
    auto kernel = which == 0 ? attention_tiles_kernel<false, 1> : which == 1 ? attention_tiles_kernel<false, 2>
                : which == 2 ? attention_tiles_kernel<true, 1> : attention_tiles_kernel<true, 2>;
    static std::atomic<bool> suffices[4];
    if (!suffices[which]) {
        cudaFuncAttributes attributes;
        const cudaError_t e = cudaFuncGetAttributes(&attributes, kernel);
        if (e != cudaSuccess) return launched(e, "e4m3_attention_tiles");
        if (!registers_suffice(attributes.numRegs)) return fail("e4m3_attention_tiles: built with other registers than its warps share out");
        suffices[which] = true;
    }
    const cudaError_t e = raise_shared_limit(kernel, bytes, raised[which]);
    if (e != cudaSuccess) return launched(e, "e4m3_attention_tiles");
    return launched(launch_kernel(g_dependent_launch != 0, kernel, dim3(n_sms), dim3(THREADS), bytes, (cudaStream_t)stream, *p, stages),
                    "e4m3_attention_tiles");
}
