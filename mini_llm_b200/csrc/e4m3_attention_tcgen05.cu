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
constexpr int SOFTMAX_WARPS = 8, CONVERTER_WARPS = 4, MMA_WARP = SOFTMAX_WARPS + CONVERTER_WARPS;
constexpr int THREADS = (MMA_WARP + 1) * 32;
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

    // Warp 0 works it out, which is the one to ask.
    __device__ explicit Schedule(const E4m3Attention& params, int n_sms) : p(params), units(0), share(0) {
        if (threadIdx.x >= 32) return;
        const int lane = threadIdx.x;
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
    uint64_t q_full, k_full[MAX_STAGES], k_empty[MAX_STAGES], v_full[MAX_STAGES], v_empty[MAX_STAGES];
    uint64_t s_ready[2], p_ready[2], o_ready[2];
    uint32_t tmem;
    int failed, more, ticket[2];
    Unit unit;
    int head;
    float q_factor[UNIT];
    float k_scale[MAX_STAGES][TILE / E4M3_BLOCK], v_scale[MAX_STAGES][TILE / E4M3_BLOCK];
    uint32_t absent[MAX_STAGES][4], none[MAX_STAGES][4];     // keys that are not there; values that are no numbers
};

__device__ __forceinline__ bool wait_or_fail(Shared& sh, uint64_t* bar, uint32_t parity) {
    return mbar_wait(bar, parity) && !*reinterpret_cast<volatile int*>(&sh.failed);
}
__device__ __forceinline__ void give_up(Shared& sh, const E4m3Attention& p, int code) {
    if (!*reinterpret_cast<volatile int*>(&sh.failed)) {
        *reinterpret_cast<volatile int*>(&sh.failed) = 1;
        atomicExch(p.status, code);
    }
}

__global__ void __launch_bounds__(THREADS, 1) attention_tiles_kernel(const E4m3Attention p, int stages, int n_sms, int* work) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ Shared sh;
    dependents_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int k_groups = (p.dim + 63) / 64, v_groups = (p.vdim + 63) / 64;
    unsigned char* tiles = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    unsigned char* q_tile = tiles;                                             // [2][k_groups]
    unsigned char* k_stage = q_tile + 2 * k_groups * GROUP_BYTES;              // [stages][k_groups]
    unsigned char* v_stage = k_stage + stages * k_groups * GROUP_BYTES;        // [stages][v_groups]
    if (threadIdx.x == 0) {
        mbar_init(&sh.q_full, CONVERTER_WARPS);
        for (int s = 0; s < MAX_STAGES; s++) {
            mbar_init(&sh.k_full[s], CONVERTER_WARPS);
            mbar_init(&sh.v_full[s], CONVERTER_WARPS);
            mbar_init(&sh.k_empty[s], 1);
            mbar_init(&sh.v_empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.s_ready[i], 1);
            mbar_init(&sh.p_ready[i], 4);
            mbar_init(&sh.o_ready[i], 1);
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
    const Schedule schedule(p, n_sms);
    // how often each barrier has been through, over all units
    int taken = 0;                                  // blocks
    uint32_t units_done = 0, s_seen[2] = {0, 0}, o_seen[2] = {0, 0};

    for (;;) {
        if (warp == 0) {
            int at = 0;
            if (lane == 0) at = atomicAdd(work, 1);
            at = __shfl_sync(0xffffffffu, at, 0);
            Unit u;
            const bool more = schedule.find(at / p.n_heads, u);
            if (lane == 0) {
                sh.more = more;
                sh.unit = u;
                sh.head = at % p.n_heads;
            }
        }
        __syncthreads();
        if (!sh.more || sh.failed) break;
        const Unit u = sh.unit;
        const int head = sh.head, kv_head = head / (p.n_heads / p.n_kv_heads);
        // blocks of each tile: the first tile's last position comes earlier
        const int last[2] = {u.pos0 + min(u.rows, TILE) - 1, u.pos0 + u.rows - 1};
        int n[2];
        n[0] = max(0, min(u.blocks, last[0] / TILE - u.block_lo + 1));
        n[1] = u.rows > TILE ? u.blocks : 0;
        if (last[0] < 0) n[0] = 0;
        if (last[1] < 0) n[1] = 0;
        const int n_blocks = max(n[0], n[1]);

        if (warp >= SOFTMAX_WARPS && warp < MMA_WARP) {
            // ---- converters: a thread a key (and two queries) ----
            const int t = threadIdx.x - SOFTMAX_WARPS * 32;
            const int* table = p.block_table + (long)u.entry * p.max_blocks;
            const int k_pieces = p.dim / 16, v_pieces = p.vdim / 16;
            struct Row {
                uint4 k[8], v[8];
                float k_scale, v_scale;
                bool there;
            } r;
            auto page_of = [&](int j) -> int {               // of this thread's key in block j; -1: it is not there
                const int key = (u.block_lo + j) * TILE + t, index = key / p.page;
                if (j >= n_blocks || key > last[1] || index >= p.max_blocks) return -1;
                const int id = table[index];
                return id < p.n_pages ? id : -1;
            };
            auto at_of = [&](int j, int id) -> long {
                const int key = (u.block_lo + j) * TILE + t;
                return ((long)id * p.n_kv_heads + kv_head) * p.page + key % p.page;
            };
            auto load_k = [&](int j, int id) {
                r.there = id >= 0;
                const long at = r.there ? at_of(j, id) : 0;
                r.k_scale = r.v_scale = 1.0f;
                if ((t & 15) == 0 && r.there) r.k_scale = p.k_scales[at / E4M3_BLOCK], r.v_scale = p.v_scales[at / E4M3_BLOCK];
                const uint4* from = reinterpret_cast<const uint4*>(p.k_pages + at * p.dim);
#pragma unroll
                for (int i = 0; i < 8; i++) r.k[i] = (r.there && i < k_pieces) ? from[i] : make_uint4(0u, 0u, 0u, 0u);
            };
            auto load_v = [&](int j, int id) {
                const bool there = id >= 0;
                const long at = there ? at_of(j, id) : 0;
                const uint4* from = reinterpret_cast<const uint4*>(p.v_pages + at * p.vdim);
#pragma unroll
                for (int i = 0; i < 8; i++) r.v[i] = (there && i < v_pieces) ? from[i] : make_uint4(0u, 0u, 0u, 0u);
            };
            // 16 codes to two 16-byte chunks of a row in a swizzled tile
            auto put = [&](unsigned char* stage, int piece, const uint4& v) {
                uint4 a, b;
                e4m3_to_half2(v.x, a.x, a.y);
                e4m3_to_half2(v.y, a.z, a.w);
                e4m3_to_half2(v.z, b.x, b.y);
                e4m3_to_half2(v.w, b.z, b.w);
                unsigned char* row = stage + (piece >> 2) * GROUP_BYTES + t * 128;
                const int c = (piece & 3) * 2;
                *reinterpret_cast<uint4*>(row + ((c ^ (t & 7)) * 16)) = a;
                *reinterpret_cast<uint4*>(row + (((c + 1) ^ (t & 7)) * 16)) = b;
            };
            int id = page_of(0), id_after = page_of(1);
            load_k(0, id);
            load_v(0, id);
            // the queries: the CTA's last unit has been read to its end (all threads have passed the barrier above)
            for (int tile = 0; tile < 2; tile++) {
                const int row = tile * TILE + t;
                const bool there = row < u.rows;
                const uint4* from = reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q) + (u.row0 + (there ? row : 0)) * p.ld_q + (long)head * p.dim);
                float top = 0.0f;
                if (there)
                    for (int i = 0; i < p.dim / 8; i++) {
                        const uint4 v = from[i];
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int c = 0; c < 4; c++) top = max_of_three(top, fabsf(__uint_as_float(w[c] << 16)), fabsf(__uint_as_float(w[c] & 0xffff0000u)));
                    }
                // (zeros, and what is not finite, stay as they are)
                const int e = top > 0.0f && top < INFINITY ? max(-110, min(110, 14 - exponent_of(top))) : 0;
                const float factor = power_of_two(e);
                sh.q_factor[row] = p.scale * power_of_two(-e) * (p.cap > 0.0f ? 1.0f : LOG2E);
                for (int i = 0; i < p.dim / 8; i++) {
                    const uint4 v = there ? from[i] : make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    uint32_t h[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) h[c] = half2_of(__uint_as_float(w[c] << 16) * factor, __uint_as_float(w[c] & 0xffff0000u) * factor);
                    *reinterpret_cast<uint4*>(q_tile + (tile * k_groups + i / 8) * GROUP_BYTES + t * 128 + (((i & 7) ^ (t & 7)) * 16)) =
                        make_uint4(h[0], h[1], h[2], h[3]);
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full);
            for (int j = 0; j < n_blocks; j++) {
                const int s = (taken + j) % stages;
                const uint32_t parity = (((taken + j) / stages) & 1) ^ 1;
                if (!__all_sync(0xffffffffu, wait_or_fail(sh, &sh.k_empty[s], parity))) {
                    give_up(sh, p, 31);
                    break;
                }
                const uint32_t absent = __ballot_sync(0xffffffffu, !r.there);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < k_pieces) put(k_stage + s * k_groups * GROUP_BYTES, i, r.k[i]);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.k_full[s]);
                const float k_scale = r.k_scale, v_scale = r.v_scale;
                const int id_now = id_after;
                id_after = page_of(j + 2);
                load_k(j + 1, id_now);
                if (!__all_sync(0xffffffffu, wait_or_fail(sh, &sh.v_empty[s], parity))) {
                    give_up(sh, p, 32);
                    break;
                }
                // (what stands beside the tiles is read until the block's P is there, which its second product waits for)
                // (a value that is no number is so in its first entry; its row is left out, and the softmax puts it back in where it is seen)
                const bool none = (r.v[0].x & 0x7fu) == 0x7fu;
                const uint32_t nones = __ballot_sync(0xffffffffu, none);
                if ((t & 15) == 0) sh.k_scale[s][t >> 4] = k_scale, sh.v_scale[s][t >> 4] = v_scale;
                if (lane == 0) sh.absent[s][warp - SOFTMAX_WARPS] = absent, sh.none[s][warp - SOFTMAX_WARPS] = nones;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < v_pieces) put(v_stage + s * v_groups * GROUP_BYTES, i, none ? make_uint4(0u, 0u, 0u, 0u) : r.v[i]);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.v_full[s]);
                load_v(j + 1, id_now);
            }
        } else if (warp == MMA_WARP) {
            // ---- products ----
            if (lane == 0 && n_blocks > 0) {
                const uint32_t idesc_s = f16_instr_desc(TILE, TILE), idesc_o = f16_instr_desc(TILE, p.vdim) | IDESC_B_MN_MAJOR;
                const int k_steps = p.dim / UMMA_K;
                auto issue_s = [&](int tile, int s) {
                    for (int kk = 0; kk < k_steps; kk++) {
                        const uint64_t a = make_smem_desc(smem_u32(q_tile + (tile * k_groups + kk / 4) * GROUP_BYTES)) + 2 * (kk % 4);
                        const uint64_t b = make_smem_desc(smem_u32(k_stage + (s * k_groups + kk / 4) * GROUP_BYTES)) + 2 * (kk % 4);
                        umma(tmem + TILE * tile, a, b, idesc_s, kk > 0 ? 1u : 0u);
                    }
                    umma_commit(&sh.s_ready[tile]);
                };
                auto issue_o = [&](int tile, int s, bool first) {
#pragma unroll
                    for (int kk = 0; kk < TILE / UMMA_K; kk++) {
                        const uint64_t b = make_smem_desc_mn(smem_u32(v_stage + s * v_groups * GROUP_BYTES + kk * 2048), GROUP_BYTES);
                        umma_from_tmem(tmem + 256 + TILE * tile, tmem + TILE * tile + kk * (UMMA_K / 2), b, idesc_o, kk > 0 || !first ? 1u : 0u);
                    }
                };
                auto stage_of = [&](int j) { return (taken + j) % stages; };
                auto parity_of = [&](int j) { return (uint32_t)(((taken + j) / stages) & 1); };
                bool ok = wait_or_fail(sh, &sh.q_full, units_done & 1) && wait_or_fail(sh, &sh.k_full[stage_of(0)], parity_of(0));
                if (ok) {
                    tcgen05_after_sync();
                    for (int tile = 0; tile < 2; tile++)
                        if (n[tile] > 0) issue_s(tile, stage_of(0));
                    umma_commit(&sh.k_empty[stage_of(0)]);
                }
                for (int j = 0; ok && j < n_blocks; j++) {
                    const int s = stage_of(j);
                    bool v_there = false, k_there = false;
                    for (int tile = 0; ok && tile < 2; tile++) {
                        if (j >= n[tile]) continue;
                        if (!v_there) ok = wait_or_fail(sh, &sh.v_full[s], parity_of(j)), v_there = true;
                        ok = ok && wait_or_fail(sh, &sh.p_ready[tile], (s_seen[tile] + j) & 1);
                        if (!ok) break;
                        tcgen05_after_sync();
                        issue_o(tile, s, j == 0);
                        if (j + 1 < n[tile]) {
                            if (!k_there) ok = wait_or_fail(sh, &sh.k_full[stage_of(j + 1)], parity_of(j + 1)), k_there = true;
                            if (!ok) break;
                            issue_s(tile, stage_of(j + 1));
                        } else {
                            umma_commit(&sh.o_ready[tile]);
                        }
                    }
                    if (!ok) break;
                    umma_commit(&sh.v_empty[s]);
                    if (j + 1 < n_blocks) umma_commit(&sh.k_empty[stage_of(j + 1)]);
                }
                if (!ok) give_up(sh, p, 33);
            }
        } else {
            // ---- softmax: a thread a row ----
            const int tile = warp >> 2, r = threadIdx.x - tile * TILE;
            const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t s_at = tmem + lane_addr + TILE * tile, o_at = tmem + lane_addr + 256 + TILE * tile;
            const int row = tile * TILE + r;
            const bool has_row = row < u.rows;
            const int pos = u.pos0 + (has_row ? row : u.rows - 1);
            const int first = p.window > 0 ? pos - p.window + 1 : 0;
            const int tile_first_pos = u.pos0 + tile * TILE;
            const bool has_cap = p.cap > 0.0f;
            const float cap_factor = has_cap ? 2.0f * LOG2E / p.cap : 0.0f, cap_log2 = p.cap * LOG2E;
            float m = -INFINITY, l = 0.0f, q_factor = 0.0f;
            bool ok = true, sees_none = false;
            for (int j = 0; j < n[tile]; j++) {
                const int s = (taken + j) % stages, key0 = (u.block_lo + j) * TILE;
                const uint32_t parity = ((taken + j) / stages) & 1;
                // (the values' barrier too: what stands beside the tiles comes with it)
                ok = wait_or_fail(sh, &sh.s_ready[tile], (s_seen[tile] + j) & 1) && wait_or_fail(sh, &sh.v_full[s], parity);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tcgen05_after_sync();
                if (j == 0) q_factor = sh.q_factor[row];
                const bool some_none = (sh.none[s][0] | sh.none[s][1] | sh.none[s][2] | sh.none[s][3]) != 0;
                const bool needs_mask = key0 + TILE - 1 > tile_first_pos || p.window > 0 || some_none ||
                                        (sh.absent[s][0] | sh.absent[s][1] | sh.absent[s][2] | sh.absent[s][3]) != 0;
                // which of 32 columns from c on this row sees
                auto seen = [&](int c) -> uint32_t {
                    const int most = pos - key0 - c, least = first - key0 - c;
                    uint32_t bits = most >= 31 ? 0xffffffffu : (most < 0 ? 0u : (2u << most) - 1u);
                    if (least > 0) bits &= least > 31 ? 0u : 0xffffffffu << least;
                    return bits & ~sh.absent[s][c >> 5];
                };
                // the row's largest, in powers of two, with the values' scale
                float top = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < TILE; c += 32) {
                    float v[32];
                    tmem_load_32(s_at + c, v);
                    if (needs_mask) {
                        const uint32_t bits = seen(c);
                        if ((sh.none[s][c >> 5] & bits) != 0) sees_none = true;
#pragma unroll
                        for (int i = 0; i < 32; i++) v[i] = (bits >> i) & 1 ? v[i] : -INFINITY;
                    }
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        float most = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 16; i += 2) most = max_of_three(most, v[16 * half + i], v[16 * half + i + 1]);
                        const float k_scale = sh.k_scale[s][c / 16 + half], t = (float)exponent_of(sh.v_scale[s][c / 16 + half]);
                        // (no factor is negative, and the cap keeps the order: the largest score is the largest product's)
                        const float y = most * (q_factor * k_scale);
                        if (most != -INFINITY) top = fmaxf(top, (has_cap ? capped(y, cap_log2, cap_factor) : y) + t);
                    }
                }
                if (__any_sync(0xffffffffu, top > m + 8.0f)) {
                    const float most = fmaxf(m, top), down = m == -INFINITY ? 0.0f : exp2_fast(m - most);
                    m = most;
                    l *= down;
                    if (j > 0) {                     // (the products into O up to here are done: S of this block came behind them)
                        for (int c = 0; c < p.vdim; c += 16) {
                            float v[16];
                            tmem_load_16(o_at + c, v);
                            uint32_t w[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) w[i] = __float_as_uint(v[i] * down);
                            tmem_store_bits_16(o_at + c, w);
                        }
                    }
                }
                const float base = (m == -INFINITY ? 0.0f : m) - 7.0f;
#pragma unroll 1
                for (int c = 0; c < TILE; c += 32) {
                    float v[32];
                    tmem_load_32(s_at + c, v);
                    const uint32_t bits = needs_mask ? seen(c) : 0xffffffffu;
                    uint32_t packed[16];
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const float v_scale = sh.v_scale[s][c / 16 + half], factor = q_factor * sh.k_scale[s][c / 16 + half];
                        const float from = (float)exponent_of(v_scale) - base;
                        float sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float x[2];
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                const float y = v[16 * half + i + e];
                                x[e] = exp2_fast(has_cap ? capped(y * factor, cap_log2, cap_factor) + from : fmaf(y, factor, from));
                                if (needs_mask && !((bits >> (16 * half + i + e)) & 1)) x[e] = 0.0f;
                                sum += x[e];
                            }
                            packed[8 * half + i / 2] = half2_of(x[0], x[1]);
                        }
                        l = fmaf(sum, 1.0f / v_scale, l);
                    }
                    // P of columns c .. c + 31 over S of columns c / 2 .. c / 2 + 15, which have been read
                    tmem_store_bits_16(s_at + c / 2, packed);
                }
                tmem_stores_landed();
                tcgen05_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_ready[tile]);
            }
            if (ok && n[tile] > 0) {
                ok = wait_or_fail(sh, &sh.o_ready[tile], o_seen[tile] & 1);
                ok = __all_sync(0xffffffffu, ok);
                tcgen05_after_sync();
            }
            if (!ok) {
                if (lane == 0) give_up(sh, p, 34);
            } else {
                if (sees_none) l = __int_as_float(0x7fffffff);
                bf16* out = static_cast<bf16*>(p.out) + (u.row0 + (has_row ? row : 0)) * p.ld_out + (long)head * p.vdim;
                const int width = (p.vdim + 63) / 64 * 64;
                bool writes = true;
                float total = l;
                float* cell = p.partial + ((long)u.cell * p.n_heads + head) * UNIT * (width + 2) + row;
                if (u.parts > 1) {
                    // this part's sums, column by column, so that the rows of a warp lie side by side
                    for (int c = 0; c < p.vdim; c += 16) {
                        float v[16];
                        if (n[tile] > 0) tmem_load_16(o_at + c, v);
#pragma unroll
                        for (int i = 0; i < 16; i++) __stcg(cell + (long)(c + i) * UNIT, n[tile] > 0 ? v[i] : 0.0f);
                    }
                    __stcg(cell + (long)width * UNIT, m);
                    __stcg(cell + (long)(width + 1) * UNIT, l);
                    __threadfence();
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + tile) : "memory");
                    int* counter = p.counters + 2 * (u.index * p.n_heads + head) + tile;
                    if (r == 0) sh.ticket[tile] = atomicAdd(counter, 1);
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + tile) : "memory");
                    writes = sh.ticket[tile] == u.parts - 1;
                    if (writes) {
                        __threadfence();
                        if (r == 0) *counter = 0;
                    }
                }
                if (writes && has_row && u.parts > 1) {
                    const long step = (long)p.n_heads * UNIT * (width + 2);
                    const float* all = cell - u.part * step;
                    float top = -INFINITY;
                    for (int q = 0; q < u.parts; q++) top = fmaxf(top, __ldcg(all + q * step + (long)width * UNIT));
                    const float anchor = top == -INFINITY ? 0.0f : top;
                    total = 0.0f;
                    for (int q = 0; q < u.parts; q++)
                        total += exp2_fast(__ldcg(all + q * step + (long)width * UNIT) - anchor) * __ldcg(all + q * step + (long)(width + 1) * UNIT);
                    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
                    for (int c = 0; c < p.vdim; c += 8) {
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) v[i] = 0.0f;
                        for (int q = 0; q < u.parts; q++) {
                            const float weight = exp2_fast(__ldcg(all + q * step + (long)width * UNIT) - anchor);
#pragma unroll
                            for (int i = 0; i < 8; i++) v[i] += weight * __ldcg(all + q * step + (long)(c + i) * UNIT);
                        }
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i] * inverse, v[2 * i + 1] * inverse);
                            w[i] = *reinterpret_cast<const uint32_t*>(&two);
                        }
                        *reinterpret_cast<uint4*>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else if (u.parts == 1) {
                    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
                    for (int c = 0; c < p.vdim; c += 16) {
                        float v[16];
                        if (n[tile] > 0) tmem_load_16(o_at + c, v);
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const __nv_bfloat162 two = n[tile] > 0 ? __floats2bfloat162_rn(v[2 * i] * inverse, v[2 * i + 1] * inverse)
                                                                   : __floats2bfloat162_rn(0.0f, 0.0f);
                            w[i] = *reinterpret_cast<const uint32_t*>(&two);
                        }
                        if (has_row) {
                            *reinterpret_cast<uint4*>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
                            *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    }
                }
                tcgen05_before_sync();
            }
        }
        // every thread counts what the barriers went through
        taken += n_blocks;
        units_done++;
        for (int i = 0; i < 2; i++) {
            s_seen[i] += n[i];
            o_seen[i] += n[i] > 0 ? 1 : 0;
        }
        __syncthreads();
        tcgen05_after_sync();
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
    const cudaError_t e = cudaFuncSetAttribute(attention_tiles_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return launched(e, "e4m3_attention_tiles");
    return launched(launch_kernel(g_dependent_launch != 0, attention_tiles_kernel, dim3(n_sms), dim3(THREADS), bytes, (cudaStream_t)stream,
                                  *p, stages, n_sms, work),
                    "e4m3_attention_tiles");
}
