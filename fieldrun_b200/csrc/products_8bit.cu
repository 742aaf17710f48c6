// Products of rows of 8-bit codes on the fifth-generation tensor core (tcgen05, kind::i8): whole numbers summed in 32 bits, scaled by
// the row's and the channel's float32 on the way out; with two weights (gate and up) the unit's activation and product on the way out, too.
//
//   out[t, f] = scale_x[t] scale_w[f] sum_k x[t, k] w[f, k]                      parts 1
//   out[t, f] = gate(g[t, f]) * u[t, f], g and u such products of two weights    parts 2
//
// Tokens are the tensor core's M: a lane of tensor memory is a token, a column a channel, so a token's gate and up of one channel
// lie in one thread, and a token's channels go out side by side.  A tile is 128 tokens of one block, or 256 of a pair of blocks
// (cta_group::2: each brings half of the channels' rows to both), by N <= 256 columns.  How many columns, and whether blocks pair, follows
// from the sizes (choose() below): the sum is exact, so nothing of the result depends on it.
//
// Blocks stay for the whole launch and take the tiles in turn.  One thread copies k-blocks (rows of 128 bytes, swizzled) of the tokens'
// and the weights' codes into a ring of stages with TMA, running ahead into the next tile; one thread issues the MMAs; the sums of a tile
// lie in one half of the tensor memory while eight warps read the other half's out.  With few tokens the weights are the traffic: their
// first stages are asked for before the kernel before this one has ended where that is safe (weights_final), and up to eight tokens are
// rounded to codes by every block for itself, into shared memory, while its first weights are on their way: one launch instead of two.
//
// Every wait on an mbarrier gives up after about a second, records a code in `status` and lets the block leave through the common exit.
#include <atomic>
#include <cmath>
#include <type_traits>

#include "products_8bit.cuh"
#include "tcgen05.cuh"

using namespace frb_tma;
using namespace frb_tc;

namespace frb_products8 {

#define P8_EPILOGUE_WARPS 8
#define P8_THREADS (64 + 32 * P8_EPILOGUE_WARPS)
#define P8_MAX_STAGES 16
#define P8_SMEM (222 * 1024)
#define P8_STAGED_BYTES (4096 * P8_EPILOGUE_WARPS)

// The gates in one form, g' sigmoid(g' (a + b g'^2)) (u' + add): silu a = 1, b = 0; tanh-gelu, 0.5 g (1 + tanh(z)) = g sigmoid(2 z) with
// z = sqrt(2 / pi) (g + 0.044715 g^3); the clamped gate a = 1.702, g' = min(g, L), u' = clamp(u, -L, L), add 1.  NaN stays NaN.  The hardware's
// exponential and reciprocal are off by 2 units in the last place each; the value is rounded to 8 bits next.  (One short form for all
// gates: 32 copies of three with exact divisions were 100 KB of instructions, and one token's unit waited 24 us for them to be fetched.)
struct Gate {
    float a, b;            // times -log2(e)
    float limit, add;      // infinity and 0 without a limit
};

struct Params {
    Lists lists;
    const float* w_scale;
    const float* x_scale;
    void* out;
    int* status;
    int rows, experts, F, FP;
    int out_stride;
    int k_blocks;
    int n;                 // channels of a tile
    int columns;           // of one tile in tensor memory: n, or 2 n with gate and up
    int x_box;             // tokens that a block copies a stage
    int n_box;             // rows of weights that a block copies a stage (in one box, or in two of gate and up)
    int per_stage;         // k-blocks of a stage
    int stages;
    int tmem_columns;
    int row_tiles;         // without lists: tiles of tokens
    int channel_tiles;
    Gate gate;
    const void* x;         // tokens as they are (kernels that round them themselves)
    int K, x_stride, whole_rows;      // their entries; from one to the next; whether every row starts on 16 bytes
    int weights_final;
    int m;                 // tokens of an MMA: 128 a block, or 64 where a tile has no more
    int staged;            // results go through shared memory
    int out_align;         // 2: rows of 32-byte multiples from a 32-byte boundary, 1: of 16, 0: neither
};

// ----------------------------------------------------------------------------- forms for one block and for a pair

template <int CTAS>
__device__ __forceinline__ void i8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CTAS == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// Instruction descriptor: 32-bit whole sums, signed 8-bit operands, both K-major.
__device__ __forceinline__ uint32_t instr_desc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// An arrival at the barrier, of a pair at both blocks' barriers, when the MMAs issued so far have finished.
template <int CTAS>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if constexpr (CTAS == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(smem_addr(bar)), "h"((uint16_t)3) : "memory");
    else
        mma_commit(bar);
}

template <int CTAS>
__device__ __forceinline__ void alloc_columns(uint32_t* slot, uint32_t columns) {
    if constexpr (CTAS == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(columns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        tmem_alloc(slot, columns);
    }
}

template <int CTAS>
__device__ __forceinline__ void free_columns(uint32_t address, uint32_t columns) {
    if constexpr (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
    else tmem_free(address, columns);
}

// The pair's first block's barrier (shared::cluster address).
__device__ __forceinline__ uint32_t first_blocks(uint64_t* bar) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_addr(bar)));
    return at;
}

// Boxes of the tokens' codes (coordinates: entry of a k-block, token, k-block) and of the weights' (entry, channel, part, k-block) into this
// block's shared memory, k-block after k-block; the bytes count on the (first) block's barrier.
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void load_tokens_box(uint32_t dst, const CUtensorMap* map, int row, int k_block, uint32_t bar) {
    if constexpr (CTAS == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(row), "r"(k_block) : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(row), "r"(k_block) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void load_weights_box(uint32_t dst, const CUtensorMap* map, int channel, int part, int k_block, uint32_t bar) {
    if constexpr (CTAS == 2)
        asm volatile(
            "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(channel), "r"(part), "r"(k_block) : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(channel), "r"(part), "r"(k_block) : "memory");
}

template <int CTAS>
__device__ __forceinline__ void everybody() {
    if constexpr (CTAS == 2) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
}

// ----------------------------------------------------------------------------- out of the kernel

__device__ __forceinline__ void load_sums(uint32_t from, uint32_t (&sums)[16]) { tmem_ld16(from, sums); }
__device__ __forceinline__ void load_sums(uint32_t from, uint32_t (&sums)[32]) {
    tmem_ld16(from, reinterpret_cast<uint32_t (&)[16]>(sums[0]));
    tmem_ld16(from + 16, reinterpret_cast<uint32_t (&)[16]>(sums[16]));
}

__device__ __forceinline__ void store_32_bytes(void* at, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// 16 neighbouring channels of a token, `left` of them inside the row.
__device__ __forceinline__ void store16(float* at, const float* v, int left, int align) {
    if (left >= 16 && align == 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[8 * h + i]);
            store_32_bytes(at + 8 * h, w);
        }
    } else if (left >= 16 && align == 1) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(at + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) if (i < left) at[i] = v[i];
    }
}
__device__ __forceinline__ void store16(bf16* at, const float* v, int left, int align) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    if (left >= 16 && align == 2) {
        store_32_bytes(at, w);
    } else if (left >= 16 && align == 1) {
        *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(at + 8) = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) if (i < left) at[i] = __float2bfloat16_rn(v[i]);
    }
}

__device__ __forceinline__ float gated(float g, float u, const Gate& gate) {
    g = g > gate.limit ? gate.limit : g;
    u = u > gate.limit ? gate.limit : u;
    u = u < -gate.limit ? -gate.limit : u;
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * fmaf(gate.b * g, g, gate.a)));
    return __fdividef(g, 1.0f + e) * (u + gate.add);
}

// The same as chunk `chunk` of a 128-byte row whose 16-byte pieces are swizzled by `swizzle`.
template <typename OutT>
__device__ __forceinline__ void put16(uint8_t* row, int chunk, int swizzle, const float* v) {
    if constexpr (sizeof(OutT) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(row + (((4 * chunk + i) ^ swizzle) << 4)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint4*>(row + (((2 * chunk + i) ^ swizzle) << 4)) =
                make_uint4(pack_bf16x2(v[8 * i], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]), pack_bf16x2(v[8 * i + 4], v[8 * i + 5]),
                           pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
    }
}

// ----------------------------------------------------------------------------- the kernel

#define P8_KEPT 8                      // runs of 8 entries of a token that a lane holds

__host__ __device__ inline int warps_a_token(int tokens) { return tokens == 1 ? 8 : tokens == 2 ? 4 : tokens <= 4 ? 2 : 1; }

// One to eight tokens rounded by the epilogue's warps: as many warps a row as there are for it.  Entry k of row r goes to k-block k / 128,
// row r of its eight of 128 bytes, the 16-byte chunk that the swizzle has there; scales to `scales`.
template <typename InT>
__device__ __forceinline__ void round_tokens(const Params& p, int ew, int lane, uint8_t* codes, float* scales, uint32_t (*tops)[P8_EPILOGUE_WARPS]) {
    const int per_row = warps_a_token(p.rows), row = ew / per_row, sub = ew % per_row;
    const bool mine = row < p.rows;
    const InT* src = (const InT*)p.x + (size_t)(mine ? row : 0) * p.x_stride;
    const int KP = p.k_blocks * FRB_8BIT_KBLOCK, step = per_row * 256;
    const int first = (sub * 32 + lane) * 8;
    Eight<InT> kept[P8_KEPT];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < P8_KEPT; ++j) {
        const int k = first + j * step;
        kept[j].clear();
        if (mine && k < p.K) kept[j].read(src + k, p.K - k, p.whole_rows);
    }
#pragma unroll
    for (int j = 0; j < P8_KEPT; ++j) top = top_of(kept[j], top);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[0][ew] = top;
    asm volatile("bar.sync 1, %0;" ::"n"(32 * P8_EPILOGUE_WARPS) : "memory");
    top = 0;
    for (int i = 0; i < per_row; ++i) top = max(top, tops[0][ew - sub + i]);
    float factor, scale;
    row_factor<InT>(top, factor, scale);
    if (!mine) return;
    const auto place = [&](int k) { return reinterpret_cast<uint2*>(codes + (k >> 7) * 1024 + row * 128 + ((((k >> 4) & 7) ^ row) << 4) + (k & 8)); };
    uint32_t again = 0;                                       // one bit for each run of eight entries that slow_codes() decides
#pragma unroll
    for (int j = 0; j < P8_KEPT; ++j) {
        const int k = first + j * step;
        if (k >= KP) break;
        bool near;
        *place(k) = codes_of(kept[j], factor, near);
        again |= (uint32_t)near << j;
    }
#pragma unroll 1
    for (int j = 0; again >> j; ++j) {
        const int k = first + j * step;
        if ((again >> j & 1) && k < p.K) *place(k) = slow_codes(src + k, p.K - k, factor, __uint_as_float(top));
    }
    if (sub == 0 && lane == 0) scales[row] = scale;
}

// InT int8_t: the tokens' codes come with the weights, stage by stage; otherwise they are rounded here (at most eight, CTAS 1, no lists).
// WHOLE: tiles of 128 tokens a block, whose results are many; without, the way out is short code in place of a fast one (one token's gated block
// of 4096 and 12288: 34.8 us with the code of whole tiles, most of it waiting for instructions, 31.9 without).
template <int CTAS, int PARTS, typename OutT, typename InT, bool WHOLE>
__global__ void __launch_bounds__(P8_THREADS, 1)
product_8bit_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ Params p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[P8_MAX_STAGES], empty_bar[P8_MAX_STAGES];
    __shared__ uint64_t sums_bar[2], read_bar[2];             // a half's sums are complete; the epilogue has read them
    __shared__ uint64_t tokens_bar;
    __shared__ uint32_t tmem_slot, token_tops[1][P8_EPILOGUE_WARPS];
    __shared__ float token_scales[8];
    __shared__ __align__(16) float w_scales[2][256];
    __shared__ int failed_flag;
    constexpr bool ROUNDS = !std::is_same<InT, int8_t>::value;
    volatile int* failed = &failed_flag;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int side = CTAS == 2 ? (int)(blockIdx.x & 1) : 0;   // which block of the pair (clusters are runs of two blocks)
    uint8_t* tokens = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);          // ROUNDS: all k-blocks of eight tokens
    uint8_t* ring = tokens + (ROUNDS ? p.k_blocks * 1024 : 0);
    // a stage: its k-blocks of tokens, then its k-blocks of weights
    const uint32_t x_bytes = (uint32_t)p.x_box * 128, w_bytes = (uint32_t)p.n_box * 128;
    const uint32_t stage_x = ROUNDS ? 0 : x_bytes * p.per_stage, stage_bytes = stage_x + w_bytes * p.per_stage;

    if (threadIdx.x == 0) {
        if (!ROUNDS) asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        for (int s = 0; s < p.stages; ++s) { bar_init(&full_bar[s], 1); bar_init(&empty_bar[s], 1); }
        for (int h = 0; h < 2; ++h) { bar_init(&sums_bar[h], 1); bar_init(&read_bar[h], P8_EPILOGUE_WARPS * CTAS); }
        bar_init(&tokens_bar, P8_EPILOGUE_WARPS);
        failed_flag = 0;
        bar_init_fence();
    }
    if (warp == 1) alloc_columns<CTAS>(&tmem_slot, (uint32_t)p.tmem_columns);
    fence_before_sync();
    everybody<CTAS>();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);

    const bool listed = p.lists.tile_expert != nullptr;
    const int items = __shfl_sync(0xffffffffu, (listed ? min(p.lists.num_tiles[0], p.lists.max_tiles) : p.row_tiles) * p.channel_tiles, 0);
    const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
    // Neighbouring items: with lists the channel tiles of one expert's rows (its weights are read once), without the tiles of tokens
    // over the same weights.
    const auto place = [&](int item, int& row0, int& expert, int& channel) {
        if (listed) {
            const int tile = item / p.channel_tiles;
            channel = (item - tile * p.channel_tiles) * p.n;
            expert = min(max(p.lists.tile_expert[tile], 0), p.experts - 1);       // (nothing is read out of place, whatever a list says)
            row0 = min(max(p.lists.tile_row0[tile], 0), p.rows);
        } else {
            const int t = item / p.row_tiles;
            channel = t * p.n;
            row0 = (item - t * p.row_tiles) * (128 * CTAS);
            expert = 0;
        }
    };

    // The whole warp goes through the loops that issue copies and MMAs, one of its lanes issues them (elect_one, tcgen05.cuh); addresses and
    // descriptors go on by additions: a stage of 8 KB costs each of the two loops more than its copies and MMAs do otherwise.
    if (warp == 0) {
        const uint32_t ring_at = smem_addr(ring), empty_at = smem_addr(empty_bar), own_full = smem_addr(full_bar);
        const uint32_t full_at = CTAS == 2 ? first_blocks(full_bar) : own_full;
        const bool by_part = CTAS == 2 && PARTS == 2;          // of a pair, the first block brings the gate's rows and the second the up's
        const int side_channel = by_part ? 0 : side * p.n_box, side_part = by_part ? side : 0;
        // (boxes that end behind the last k-block are filled with zeros there)
        const auto load_weights = [&](int s, int k_block, int part, int channel) {
            if (side == 0) expect_bytes(own_full + 8 * s, stage_bytes * CTAS);
            load_weights_box<CTAS>(ring_at + s * stage_bytes + stage_x, &map_w, channel, part, k_block, full_at + 8 * s);
        };
        // The first stages' weights before the wait for the tokens' codes, then their tokens, then stage after stage.
        int row0, expert, channel, ahead = 0;
        if (!p.weights_final) wait_for_previous_kernel();
        for (int item = first; item < items && ahead < p.stages; item += step) {
            place(item, row0, expert, channel);
            for (int k = 0; k < p.k_blocks && ahead < p.stages; k += p.per_stage, ++ahead)
                if (elect_one()) load_weights(ahead, k, expert * PARTS + side_part, channel + side_channel);
        }
        __syncwarp();
        wait_for_previous_kernel();
        let_next_kernel_start();
        int issued = 0, s = 0;
        uint32_t parity = 1;                                   // of the phase in which the stage's earlier use was given back
        bool ok = true;
        for (int item = first; item < items && ok; item += step) {
            place(item, row0, expert, channel);
            const int part = expert * PARTS + side_part, from = channel + side_channel, token = row0 + side * 128;
            for (int k = 0; k < p.k_blocks; k += p.per_stage) {
                if (issued >= ahead) {
                    if (!bar_try(empty_at + 8 * s, parity) && !warp_wait(&empty_bar[s], parity, failed)) {
                        if (lane == 0) atomicExch(p.status, 121);
                        ok = false;
                        break;
                    }
                    if (elect_one()) load_weights(s, k, part, from);
                }
                if (!ROUNDS && elect_one()) load_tokens_box<CTAS>(ring_at + s * stage_bytes, &map_x, token, k, full_at + 8 * s);
                ++issued;
                if (++s == p.stages) { s = 0; parity ^= 1; }
            }
        }
        __syncwarp();
        if (lane == 0) {
            // every stage has come back before the block may leave (a pair's first block signals this one's barriers)
            for (int back = 0; back < p.stages && back < issued; ++back) {
                const int q = issued - 1 - back;
                if (ok) {
                    if (!bar_wait(&empty_bar[q % p.stages], (uint32_t)((q / p.stages) & 1), failed)) { atomicExch(p.status, 122); ok = false; }
                } else if (side == 0) {                       // copies may still be on their way: a bounded time for each to land
                    int again = 0;
                    bar_wait(&full_bar[q % p.stages], (uint32_t)((q / p.stages) & 1), &again, 20000000ll);
                }
            }
        }
    } else if (warp == 1) {
        if (side == 0) {
            wait_for_previous_kernel();                       // no tokens before that; the limits of the waits below are for this kernel's own work
            const uint32_t idesc = instr_desc_i8(p.m * CTAS, p.columns);
            const uint64_t first_x = tile_desc(smem_addr(ROUNDS ? tokens : ring)), first_w = tile_desc(smem_addr(ring) + stage_x);
            const uint32_t stage_step = stage_bytes >> 4, x_step = ROUNDS ? 64 : x_bytes >> 4, w_step = w_bytes >> 4;      // in 16 bytes
            int s = 0, half = 0;
            uint32_t parity = 0, read_parity = 3;             // (one bit of the latter for each half)
            bool ok = true;
            if (ROUNDS && first < items && !warp_wait(&tokens_bar, 0, failed)) { if (lane == 0) atomicExch(p.status, 126); ok = false; }
            for (int item = first; item < items && ok; item += step) {
                if (!warp_wait(&read_bar[half], (read_parity >> half) & 1, failed)) { if (lane == 0) atomicExch(p.status, 123); break; }
                read_parity ^= 1u << half;
                fence_after_sync();
                const uint32_t sums = tmem + half * p.columns;
                uint32_t add = 0;                             // 0: the item's first MMA sets the sums
                for (int left = p.k_blocks, at = 0; left > 0; left -= p.per_stage, at += p.per_stage) {
                    if (!warp_wait(&full_bar[s], parity, failed)) { if (lane == 0) atomicExch(p.status, 124); ok = false; break; }
                    fence_after_sync();
                    if (elect_one()) {
                        uint64_t desc_x = first_x + (ROUNDS ? at * 64 : s * stage_step), desc_w = first_w + s * stage_step;
                        const int blocks = min(p.per_stage, left);
                        for (int b = 0; b < blocks; ++b, desc_x += x_step, desc_w += w_step) {
#pragma unroll
                            for (int k = 0; k < FRB_8BIT_KBLOCK / 32; ++k, add = 1)           // 32 k per MMA: 32 bytes along the swizzled row
                                i8_mma<CTAS>(sums, desc_x + 2 * k, desc_w + 2 * k, idesc, add);
                        }
                        commit<CTAS>(&empty_bar[s]);
                        if (left <= p.per_stage) commit<CTAS>(&sums_bar[half]);
                    }
                    add = 1;
                    __syncwarp();
                    if (++s == p.stages) { s = 0; parity ^= 1; }
                }
                half ^= 1;
            }
        }
    } else {
        // Warp w may read the 32 lanes of tensor memory that are numbered by w & 3; the two warps of a quarter take the groups of 16
        // channels in turn.
        const int quarter = warp & 3, turn = (warp - 2) >> 2, span = p.m >> 2;               // (64 tokens lie in the first 16 lanes of each quarter)
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        OutT* out = (OutT*)p.out;
        wait_for_previous_kernel();
        let_next_kernel_start();
        if (ROUNDS) {
            if constexpr (ROUNDS) round_tokens<InT>(p, warp - 2, lane, tokens, token_scales, token_tops);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // the tensor core reads what was written here
            __syncwarp();
            if (lane == 0) bar_arrive(&tokens_bar);
            asm volatile("bar.sync 1, %0;" ::"n"(32 * P8_EPILOGUE_WARPS) : "memory");       // the scales are there
        }
        // Staged results: a warp's 32 tokens by 128 bytes of channels go through a buffer of its own (16-byte pieces swizzled by the token) and from
        // there in whole lines; otherwise every lane stores its token's channels.  (8,192 tokens, 1024 x 8192, float32: 109 us without.  Copies by TMA,
        // with their fence, wait and map, took 92.)
        // A step is 32 channels, or 16 of gate and up.
        constexpr int STEP = PARTS == 1 && WHOLE ? 32 : 16, HALVES = WHOLE ? 2 : 1, GROUP_STEPS = 128 / (int)sizeof(OutT) / STEP;        // steps in 128 bytes
        const bool staged = WHOLE && p.staged;
        const int shift = staged ? (GROUP_STEPS == 1 ? 0 : 1) : 0;
        uint8_t* buffer = ring + (size_t)p.stages * stage_bytes + (warp - 2) * 4096;
        const auto step_at = [&](int i) { return STEP * ((((i >> shift) * 2 + turn) << shift) + (i & ((1 << shift) - 1))); };
        int half = 0;
        uint32_t sums_parity = 0;                                 // one bit for each half
        // A tile's place and scales are read while the one before it is computed.
        float next_x = 0.f, next_w = 0.f;
        int next_row0 = 0, next_channel = 0, next_rows = 0;
        const auto ask = [&](int item) {
            if (item >= items) return;
            int expert;
            place(item, next_row0, expert, next_channel);
            next_rows = listed ? min(p.lists.tile_rows, min(p.lists.offsets[expert + 1], p.rows) - next_row0) : p.rows - next_row0;
            const int within = side * 128 + quarter * span + lane, i = threadIdx.x - 64;
            if (!ROUNDS && within < next_rows && lane < span && quarter * span + lane < p.x_box) next_x = p.x_scale[next_row0 + within];
            if (i < p.columns) {
                const int part = PARTS == 2 && i >= p.n ? 1 : 0, c = i - part * p.n;
                next_w = next_channel + c < p.F ? p.w_scale[((size_t)expert * PARTS + part) * p.FP + next_channel + c] : 0.f;
            }
        };
        ask(first);
        for (int item = first; item < items; item += step) {
            const int row0 = next_row0, channel = next_channel, rows = next_rows;
            const int warp_row = side * 128 + quarter * span, within = warp_row + lane;
            const bool mine = within < rows && lane < span && quarter * span + lane < p.x_box;
            const bool any = warp_row < rows && quarter * span < p.x_box;
            const int row = row0 + within;
            // A sum times the token's scale times the channel's; a token's scale of one and more (or NaN) comes last, in a branch that hardly ever is
            // taken, so that no product on the way leaves float32's range where the result does not (scales are 2^-103 and more, sums below 2^31).
            // With gate and up the channel's scale always comes first (the branch's instructions cost one token's block 1.4 us of 34): the
            // same for channels' scales below 2^96.
            const float x_scale = !mine ? 0.f : ROUNDS ? token_scales[within & 7] : next_x;
            const float x_first = x_scale < 1.f ? x_scale : 1.f, x_last = x_scale < 1.f ? 1.f : x_scale;
            const bool large = __any_sync(0xffffffffu, !(x_scale < 1.f));
            const int channels = min(p.n, p.F - channel);
            float* scales = w_scales[half];
            scales[threadIdx.x - 64] = next_w;                        // (there are as many threads as columns at most)
            ask(item + step);
            asm volatile("bar.sync 1, %0;" ::"n"(32 * P8_EPILOGUE_WARPS) : "memory");
            // (a warp whose wait ran out goes through the other items without work: all warps meet at the barrier above)
            const bool done = __all_sync(0xffffffffu, bar_wait(&sums_bar[half], (sums_parity >> half) & 1, failed));
            if (!done && lane == 0) atomicExch(p.status, 125);
            sums_parity ^= 1u << half;
            fence_after_sync();
            if (any && done) {
                const uint32_t sums = lanes + half * p.columns;
                OutT* dst = out + (size_t)row * p.out_stride + channel;
                uint32_t acc[HALVES][PARTS][STEP];                 // (two: the next step's sums come while this one's are scaled)
                if (HALVES == 2 && step_at(0) < channels) {
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) load_sums(sums + q * p.n + step_at(0), acc[0][q]);
                }
#pragma unroll 1
                for (int turns = 0; step_at(turns) < channels; turns += HALVES) {
#pragma unroll
                    for (int h = 0; h < HALVES; ++h) {
                        const int c0 = step_at(turns + h), next = step_at(turns + h + 1);
                        if (c0 >= channels) break;
                        if (HALVES == 1) {
#pragma unroll
                            for (int q = 0; q < PARTS; ++q) load_sums(sums + q * p.n + c0, acc[0][q]);
                        }
                        tmem_wait_ld();
                        if (HALVES == 2 && next < channels) {
#pragma unroll
                            for (int q = 0; q < PARTS; ++q) load_sums(sums + q * p.n + next, acc[HALVES - 1 - h][q]);
                        }
                        float v[STEP];
#pragma unroll
                        for (int i = 0; i < STEP; i += 4) {
                            const float4 s0 = *reinterpret_cast<const float4*>(scales + c0 + i), s1 = *reinterpret_cast<const float4*>(scales + (PARTS - 1) * p.n + c0 + i);
                            const float first_scale[4] = {s0.x, s0.y, s0.z, s0.w}, second_scale[4] = {s1.x, s1.y, s1.z, s1.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                if (PARTS == 1) {
                                    v[i + j] = (float)(int)acc[h][0][i + j] * x_first * first_scale[j];
                                    if (large) v[i + j] *= x_last;
                                } else {
                                    v[i + j] = gated((float)(int)acc[h][0][i + j] * first_scale[j] * x_scale,
                                                     (float)(int)acc[h][PARTS - 1][i + j] * second_scale[j] * x_scale, p.gate);
                                }
                            }
                        }
                        if (!staged) {
#pragma unroll
                            for (int i = 0; i < STEP; i += 16)
                                if (mine && c0 + i < channels) store16(dst + c0 + i, v + i, channels - c0 - i, p.out_align);
                            continue;
                        }
                        const int in_group = (turns + h) & (GROUP_STEPS - 1);
#pragma unroll
                        for (int i = 0; i < STEP; i += 16) put16<OutT>(buffer + lane * 128, in_group * (STEP / 16) + i / 16, lane & 7, v + i);
                        if (in_group == GROUP_STEPS - 1 || next >= channels) {
                            __syncwarp();
                            const int piece = lane & 7, from = c0 - STEP * in_group + piece * (16 / (int)sizeof(OutT));
                            uint4 w[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {             // four tokens at a time, 128 bytes of each
                                const int r = 4 * i + (lane >> 3);
                                w[i] = *reinterpret_cast<const uint4*>(buffer + r * 128 + ((piece ^ (r & 7)) << 4));
                            }
                            __syncwarp();
                            OutT* to = out + (size_t)(row0 + warp_row + (lane >> 3)) * p.out_stride + channel + from;
#pragma unroll
                            for (int i = 0; i < 8; ++i, to += 4 * (size_t)p.out_stride)
                                if (warp_row + 4 * i + (lane >> 3) < rows && from < channels) *reinterpret_cast<uint4*>(to) = w[i];
                        }
                    }
                }
                tmem_wait_ld();
            }
            fence_before_sync();
            __syncwarp();
            if (lane == 0) {                                  // this warp has what it needs of this half
                if (CTAS == 2) {
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(first_blocks(&read_bar[half])) : "memory");
                } else {
                    bar_arrive(&read_bar[half]);
                }
            }
            half ^= 1;
        }
    }
    __syncwarp();
    fence_before_sync();
    everybody<CTAS>();
    fence_after_sync();
    if (warp == 1) free_columns<CTAS>(tmem, (uint32_t)p.tmem_columns);
}

// ----------------------------------------------------------------------------- host side

static bool map_of(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    EncodeFn fn = encoder();
    cuuint32_t elem[4] = {1, 1, 1, 1};
    return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of codes as (entry of a k-block, row, k-block), `box_rows` rows and `blocks` k-blocks a box.
static bool map_tokens(CUtensorMap* map, const void* base, uint64_t rows, uint64_t KP, uint32_t box_rows, uint32_t blocks) {
    const cuuint64_t dims[3] = {128, rows, KP / 128}, strides[2] = {KP, 128};
    const cuuint32_t box[3] = {128, box_rows, blocks};
    return map_of(map, base, 3, dims, strides, box);
}

// Weights as (entry of a k-block, channel, part of any expert, k-block).
static bool map_weights(CUtensorMap* map, const void* base, uint64_t parts, uint64_t FP, uint64_t KP, uint32_t box_rows, uint32_t box_parts, uint32_t blocks) {
    const cuuint64_t dims[4] = {128, FP, parts, KP / 128}, strides[3] = {KP, FP * KP, 128};
    const cuuint32_t box[4] = {128, box_rows, box_parts, blocks};
    return map_of(map, base, 4, dims, strides, box);
}

// Whether the product rounds the tokens itself: up to eight that the warps hold in registers, and whose codes leave half of a block's
// shared memory to the weights.  (Longer ones would be read twice, 10 us for eight tokens of 4,096 entries where a launch costs 3.)
bool tokens_fit(int rows, int K) { return rows <= 8 && K <= 14336 && K <= warps_a_token(rows) * P8_KEPT * 256; }

// Tokens that a block copies at a time: 128, or as many as a tile has where that is less.
static int tokens_box(const Product& p, int ctas) {
    const int tile = p.lists.tile_expert ? p.lists.tile_rows : p.rows;
    return ctas == 2 || tile >= 128 ? 128 : up_to(tile, 8);
}

struct Shape { int ctas, n, per_stage, stages; };

// The form of a tile and of a stage: the one whose last block is done first.  Clocks of a k-block: the tensor core's 2 a column, but at
// least one a row of its M (it reads 64 or 128 tokens' codes from shared memory, however many there are), or those of the copies at 45 bytes a clock and SM;
// of a stage at least 350 (the round from one copy to the next through both barriers); of a tile some 500 besides.  A stage is 52 KB at most
// and holds several k-blocks where tiles are narrow: a box of them reads runs of several hundred bytes of a row at once.  Measured with a
// 4096 x 24576 weight and one token, us: 32 channels and 1 k-block 56, 2 41, 8 30; 48 and 8 23; 64 and 4 23; 96 and 1 27, 4 22; 128 and 2 25.
static Shape choose(const Product& p, int sms) {
    const int k_blocks = up_to(p.K, FRB_8BIT_KBLOCK) / FRB_8BIT_KBLOCK;
    const bool listed = p.lists.tile_expert, rounds = !p.x_scale;
    Shape best = {};
    double best_cost = 1e300;
    for (int ctas = 1; ctas <= 2; ++ctas) {
        if (listed ? (p.lists.tile_rows > 128) != (ctas == 2) : ctas == 2 && p.rows <= 128) continue;
        const long long row_tiles = listed ? p.lists.max_tiles : (p.rows + 128 * ctas - 1) / (128 * ctas);
        const int x_box = tokens_box(p, ctas), x_rows = rounds ? 0 : x_box, m = x_box <= 64 ? 64 : 128;
        const int ring = P8_SMEM - 1024 - (x_box < 128 ? m * 128 : P8_STAGED_BYTES) - (rounds ? k_blocks * 1024 : 0);
        for (int n = 16 * ctas; n * p.parts <= 256; n += 16 * ctas) {
            const int columns = n * p.parts, block = (x_rows + columns / ctas) * 128;
            int per_stage = 1;
            while (per_stage < 16 && per_stage < k_blocks && 2 * per_stage * block <= 52 * 1024 && 3 * 2 * per_stage * block <= ring) per_stage *= 2;
            const int fit = ring / (block * per_stage), stages = fit < P8_MAX_STAGES ? fit : P8_MAX_STAGES;
            if (stages < 2) continue;
            const double math = 2.0 * columns > m ? 2.0 * columns : m, feed = block / 45.0, both = per_stage * (math > feed ? math : feed);
            const long long items = row_tiles * ((p.F + n - 1) / n), workers = sms / ctas;
            const double cost = (double)((items + workers - 1) / workers) * ((k_blocks + per_stage - 1) / per_stage * (both > 350.0 ? both : 350.0) + 500.0) +
                                8.0 * columns;
            if (cost < best_cost) { best_cost = cost; best = {ctas, n, per_stage, stages}; }
            if (n >= p.F) break;
        }
    }
    return best;
}

// Lets a kernel have a block's whole shared memory: asked for once a kernel and device.
template <auto KERNEL>
static void may_have_shared() {
    static std::atomic<unsigned> asked{0};
    int device = 0;
    cudaGetDevice(&device);
    const unsigned bit = 1u << (device & 31);
    if (asked.load(std::memory_order_relaxed) & bit) return;
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, P8_SMEM) == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
}

int product(const Product& q, cudaStream_t stream) {
    if (q.rows == 0 || (q.lists.tile_expert && q.lists.max_tiles == 0)) return 0;
    const int KP = up_to(q.K, FRB_8BIT_KBLOCK), FP = up_to(q.F, FRB_8BIT_ROWS);
    FRB_CHECK_ARG(q.K >= 1 && q.K <= FRB_8BIT_MOST_INNER, "product in 8 bits: an inner size of %d is outside 1..%d", q.K, FRB_8BIT_MOST_INNER);
    FRB_CHECK_ARG(q.F >= 1 && q.experts >= 1 && (q.parts == 1 || q.parts == 2), "product in 8 bits: %d experts of %d x %d channels", q.experts, q.parts, q.F);
    FRB_CHECK_ARG((((uintptr_t)q.w | (q.x_scale ? (uintptr_t)q.x : 0) | (uintptr_t)q.w_scale) & 15) == 0, "product in 8 bits: codes and scales start on 16 bytes");
    FRB_CHECK_ARG(!q.lists.tile_expert || (q.lists.tile_rows >= 1 && q.lists.tile_rows <= 128) || q.lists.tile_rows == 256,
                  "product in 8 bits: tiles of %d rows (at most 128, or 256)", q.lists.tile_rows);
    FRB_CHECK_ARG(q.F < (1 << 30) && q.rows < (1 << 30) && q.experts < (1 << 30), "product in 8 bits: %d rows of %d channels and %d experts exceed a tensor map",
                  q.rows, q.F, q.experts);
    const int sms = frb_sm_count();
    const bool rounds = !q.x_scale;
    FRB_CHECK_ARG(!rounds || (tokens_fit(q.rows, q.K) && !q.lists.tile_expert), "product in 8 bits: %d tokens of %d entries to round", q.rows, q.K);
    const Shape shape = choose(q, sms);
    const int ctas = shape.ctas;
    FRB_CHECK_ARG(ctas != 0, "product in 8 bits: no form for %d rows of %d entries", q.rows, q.K);
    Params p;
    p.lists = q.lists; p.w_scale = q.w_scale; p.x_scale = q.x_scale; p.out = q.out; p.status = q.status;
    p.rows = q.rows; p.experts = q.experts; p.F = q.F; p.FP = FP; p.k_blocks = KP / FRB_8BIT_KBLOCK; 
    const float log2e = 1.4426950408889634f, slope = q.limit > 0.f ? FRB_CLAMPED_GATE_SLOPE : q.gate == FRB_GATE_GELU_TANH ? 1.5957691216057308f : 1.0f;
    p.gate.a = -log2e * slope;
    p.gate.b = q.limit <= 0.f && q.gate == FRB_GATE_GELU_TANH ? -log2e * slope * 0.044715f : 0.f;
    p.gate.limit = q.limit > 0.f ? q.limit : INFINITY;
    p.gate.add = q.limit > 0.f ? 1.f : 0.f;
    p.n = shape.n;
    p.columns = p.n * q.parts;
    p.x_box = tokens_box(q, ctas);
    p.n_box = p.columns / ctas;
    p.m = p.x_box <= 64 ? 64 : 128;
    // (steps of 32 columns may read behind the second half's last)
    const int two = p.columns + up_to(p.columns, 32);
    p.tmem_columns = two <= 32 ? 32 : two <= 64 ? 64 : two <= 128 ? 128 : two <= 256 ? 256 : 512;
    p.per_stage = shape.per_stage;
    p.stages = shape.stages;
    // the A operand of an MMA is 64 or 128 rows, whatever was copied: the last stage's has to end inside the block's shared memory
    const size_t smem = 1024 + (rounds ? p.k_blocks * 1024 : 0) + (size_t)p.stages * p.per_stage * ((rounds ? 0 : p.x_box) + p.n_box) * 128 +
                        (p.x_box < 128 ? p.m * 128 : P8_STAGED_BYTES);
    FRB_CHECK_ARG(p.stages >= 2 && p.stages <= P8_MAX_STAGES && smem <= P8_SMEM, "product in 8 bits: %d stages in %zu bytes", p.stages, smem);
    p.x = q.x; p.K = q.K; p.x_stride = q.x_stride; p.weights_final = q.weights_final;
    p.whole_rows = q.x_stride % 8 == 0 && ((uintptr_t)q.x & 15) == 0;
    p.row_tiles = (q.rows + 128 * ctas - 1) / (128 * ctas);
    p.channel_tiles = (q.F + p.n - 1) / p.n;
    const long long most = (long long)(q.lists.tile_expert ? q.lists.max_tiles : p.row_tiles) * p.channel_tiles;
    FRB_CHECK_ARG(most < (1ll << 31) - 4096, "product in 8 bits: %d rows of %d channels exceed the count of tiles", q.rows, q.F);
    const int row_bytes = q.out_stride * (q.out_type == FRB_F32 ? 4 : 2);
    p.out_stride = q.out_stride;
    p.out_align = row_bytes % 32 == 0 && ((uintptr_t)q.out & 31) == 0 ? 2 : row_bytes % 16 == 0 && ((uintptr_t)q.out & 15) == 0 ? 1 : 0;
    // tiles of 128 tokens go out through shared memory where the results' rows are multiples of 16 bytes and tiles end with 128 bytes
    p.staged = p.x_box == 128 && p.out_align >= 1 && p.n % (q.out_type == FRB_F32 ? 32 : 64) == 0;
    CUtensorMap map_x, map_w;
    const int box_parts = ctas == 2 ? 1 : q.parts;
    FRB_CHECK_ARG((rounds || map_tokens(&map_x, q.x, q.rows, KP, p.x_box, p.per_stage)) &&
                      map_weights(&map_w, q.w, (uint64_t)q.experts * q.parts, FP, KP, p.n_box / box_parts, box_parts, p.per_stage),
                  "product in 8 bits: cuTensorMapEncodeTiled failed or is not available");
    const long long workers = sms / ctas;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)((most < workers ? most : workers) * ctas));
    config.blockDim = dim3(P8_THREADS);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    config.attrs = attributes;
    if (ctas == 2) {
        cudaLaunchAttribute& pairs = attributes[config.numAttrs++];
        pairs.id = cudaLaunchAttributeClusterDimension;
        pairs.val.clusterDim.x = 2;
        pairs.val.clusterDim.y = pairs.val.clusterDim.z = 1;
    }
    if ((long)config.gridDim.x <= frb_dependent_launch_blocks()) {
        cudaLaunchAttribute& early = attributes[config.numAttrs++];
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
    }
#define LAUNCH(CTAS, PARTS, OutT, InT, WHOLE)                                                                                         \
    do {                                                                                                                              \
        may_have_shared<product_8bit_kernel<CTAS, PARTS, OutT, InT, WHOLE>>();                                                         \
        cudaLaunchKernelEx(&config, product_8bit_kernel<CTAS, PARTS, OutT, InT, WHOLE>, map_x, map_w, p);                             \
    } while (0)
    FRB_CHECK_ARG(q.parts == 1 || q.out_type == FRB_F32, "product in 8 bits: gated units come out in float32");
    if (q.parts == 2) {
        if (rounds) { FRB_DISPATCH_DTYPE(q.x_type, InT, LAUNCH(1, 2, float, InT, false)); }
        else if (ctas == 2) LAUNCH(2, 2, float, int8_t, true);
        else if (p.x_box == 128) LAUNCH(1, 2, float, int8_t, true);
        else LAUNCH(1, 2, float, int8_t, false);
    } else {
        FRB_DISPATCH_DTYPE(q.out_type, OutT, {
            if (rounds) { FRB_DISPATCH_DTYPE(q.x_type, InT, LAUNCH(1, 1, OutT, InT, false)); }
            else if (ctas == 2) LAUNCH(2, 1, OutT, int8_t, true);
            else if (p.x_box == 128) LAUNCH(1, 1, OutT, int8_t, true);
            else LAUNCH(1, 1, OutT, int8_t, false);
        });
    }
#undef LAUNCH
    FRB_RETURN_LAUNCH("product_8bit");
}

}  // namespace frb_products8
