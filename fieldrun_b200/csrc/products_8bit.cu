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
// first stages are asked for before the kernel before this one has ended (it makes the tokens' codes; whatever wrote weights or lists had
// ended before that one let this one start).
//
// Every wait on an mbarrier gives up after about a second, records a code in `status` and lets the block leave through the common exit.
#include "products_8bit.cuh"
#include "tcgen05.cuh"

using namespace frb_tma;
using namespace frb_tc;

namespace frb_products8 {

#define P8_EPILOGUE_WARPS 8
#define P8_THREADS (64 + 32 * P8_EPILOGUE_WARPS)
#define P8_MAX_STAGES 16
#define P8_SMEM (220 * 1024)

struct Params {
    Lists lists;
    const float* w_scale;
    const float* x_scale;
    void* out;
    int* status;
    int rows, F, FP;
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
    int gate;
    float limit;
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

// A box into this block's shared memory; the bytes count on the (first) block's barrier.
template <int CTAS>
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CTAS == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(smem_addr(dst)), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(smem_addr(dst)), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
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

__device__ __forceinline__ void store_32_bytes(void* at, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// 16 neighbouring channels of a token, `left` of them inside the row.
__device__ __forceinline__ void store16(float* at, const float (&v)[16], int left, int align) {
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
__device__ __forceinline__ void store16(bf16* at, const float (&v)[16], int left, int align) {
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

__device__ __forceinline__ float gated(float g, float u, int gate, float limit) {
    if (limit <= 0.f && gate == FRB_GATE_GELU_TANH)
        return 0.5f * g * (1.0f + tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g))) * u;
    return paired_gate(g, u, limit);
}

// ----------------------------------------------------------------------------- the kernel

template <int CTAS, int PARTS, typename OutT>
__global__ void __launch_bounds__(P8_THREADS, 1)
product_8bit_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ Params p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[P8_MAX_STAGES], empty_bar[P8_MAX_STAGES];
    __shared__ uint64_t sums_bar[2], read_bar[2];             // a half's sums are complete; the epilogue has read them
    __shared__ uint32_t tmem_slot;
    __shared__ int failed_flag;
    volatile int* failed = &failed_flag;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int side = CTAS == 2 ? (int)(blockIdx.x & 1) : 0;   // which block of the pair (clusters are runs of two blocks)
    uint8_t* ring = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t x_bytes = (uint32_t)p.x_box * 128, block_bytes = x_bytes + (uint32_t)p.n_box * 128;
    const uint32_t stage_bytes = block_bytes * p.per_stage;

    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        for (int s = 0; s < p.stages; ++s) { bar_init(&full_bar[s], 1); bar_init(&empty_bar[s], 1); }
        for (int h = 0; h < 2; ++h) { bar_init(&sums_bar[h], 1); bar_init(&read_bar[h], P8_EPILOGUE_WARPS * CTAS); }
        failed_flag = 0;
        bar_init_fence();
    }
    if (warp == 1) alloc_columns<CTAS>(&tmem_slot, (uint32_t)p.tmem_columns);
    fence_before_sync();
    everybody<CTAS>();
    fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);

    const bool listed = p.lists.tile_expert != nullptr;
    const int items = __shfl_sync(0xffffffffu, (listed ? p.lists.num_tiles[0] : p.row_tiles) * p.channel_tiles, 0);
    const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
    // Neighbouring items: with lists the channel tiles of one expert's rows (its weights are read once), without the tiles of tokens
    // over the same weights.
    const auto place = [&](int item, int& row0, int& expert, int& channel) {
        if (listed) {
            const int tile = item / p.channel_tiles;
            channel = (item - tile * p.channel_tiles) * p.n;
            expert = p.lists.tile_expert[tile];
            row0 = p.lists.tile_row0[tile];
        } else {
            const int t = item / p.row_tiles;
            channel = t * p.n;
            row0 = (item - t * p.row_tiles) * (128 * CTAS);
            expert = 0;
        }
    };
    const int stages_per_item = (p.k_blocks + p.per_stage - 1) / p.per_stage;

    if (warp == 0) {
        if (lane == 0) {
            const auto barrier_at = [&](int s) { return CTAS == 2 ? first_blocks(&full_bar[s]) : smem_addr(&full_bar[s]); };
            const auto load_weights = [&](int s, int st, int expert, int channel) {
                const int blocks = min(p.per_stage, p.k_blocks - st * p.per_stage);
                if (side == 0) bar_expect(&full_bar[s], block_bytes * blocks * CTAS);
                const uint32_t bar = barrier_at(s);
                const int row = (expert * PARTS) * p.FP + channel;
                for (int b = 0; b < blocks; ++b) {
                    uint8_t* dst = ring + (size_t)s * stage_bytes + b * block_bytes + x_bytes;
                    const int k = (st * p.per_stage + b) * FRB_8BIT_KBLOCK;
                    if (PARTS == 1) load_box<CTAS>(dst, &map_w, k, row + side * p.n_box, bar);
                    else if (CTAS == 2) load_box<CTAS>(dst, &map_w, k, row + side * p.FP, bar);
                    else { load_box<CTAS>(dst, &map_w, k, row, bar); load_box<CTAS>(dst + p.n * 128, &map_w, k, row + p.FP, bar); }
                }
            };
            const auto load_tokens = [&](int s, int st, int row0) {
                const int blocks = min(p.per_stage, p.k_blocks - st * p.per_stage);
                const uint32_t bar = barrier_at(s);
                for (int b = 0; b < blocks; ++b)
                    load_box<CTAS>(ring + (size_t)s * stage_bytes + b * block_bytes, &map_x, (st * p.per_stage + b) * FRB_8BIT_KBLOCK,
                                   row0 + side * 128, bar);
            };
            // The first stages' weights before the wait for the tokens' codes, then their tokens, then stage after stage.
            int row0, expert, channel, ahead = 0;
            for (int item = first; item < items && ahead < p.stages; item += step) {
                place(item, row0, expert, channel);
                for (int st = 0; st < stages_per_item && ahead < p.stages; ++st) load_weights(ahead++, st, expert, channel);
            }
            wait_for_previous_kernel();
            let_next_kernel_start();
            int issued = 0, s = 0;
            uint32_t parity = 1;                              // of the phase in which the stage's earlier use was given back
            bool ok = true;
            for (int item = first; item < items && ok; item += step) {
                place(item, row0, expert, channel);
                for (int st = 0; st < stages_per_item; ++st) {
                    if (issued >= ahead) {
                        if (!bar_wait(&empty_bar[s], parity, failed)) { atomicExch(p.status, 121); ok = false; break; }
                        load_weights(s, st, expert, channel);
                    }
                    load_tokens(s, st, row0);
                    ++issued;
                    if (++s == p.stages) { s = 0; parity ^= 1; }
                }
            }
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
            const uint32_t idesc = instr_desc_i8(128 * CTAS, p.columns), ring_at = smem_addr(ring);
            int s = 0, half = 0;
            uint32_t parity = 0, read_parity = 3;             // (one bit of the latter for each half)
            bool ok = true;
            for (int item = first; item < items && ok; item += step) {
                if (!warp_wait(&read_bar[half], (read_parity >> half) & 1, failed)) { if (lane == 0) atomicExch(p.status, 123); break; }
                read_parity ^= 1u << half;
                fence_after_sync();
                const uint32_t sums = tmem + half * p.columns;
                for (int st = 0; st < stages_per_item; ++st) {
                    if (!warp_wait(&full_bar[s], parity, failed)) { if (lane == 0) atomicExch(p.status, 124); ok = false; break; }
                    fence_after_sync();
                    const int blocks = min(p.per_stage, p.k_blocks - st * p.per_stage);
                    if (elect_one()) {
                        for (int b = 0; b < blocks; ++b) {
                            const uint64_t desc_x = tile_desc(ring_at + s * stage_bytes + b * block_bytes);
                            const uint64_t desc_w = tile_desc(ring_at + s * stage_bytes + b * block_bytes + x_bytes);
#pragma unroll
                            for (int k = 0; k < FRB_8BIT_KBLOCK / 32; ++k)           // 32 k per MMA: 32 bytes along the swizzled row
                                i8_mma<CTAS>(sums, desc_x + 2 * k, desc_w + 2 * k, idesc, (st | b | k) != 0);
                        }
                        commit<CTAS>(&empty_bar[s]);
                        if (st == stages_per_item - 1) commit<CTAS>(&sums_bar[half]);
                    }
                    __syncwarp();
                    if (++s == p.stages) { s = 0; parity ^= 1; }
                }
                half ^= 1;
            }
        }
    } else {
        // Warp w may read the 32 lanes of tensor memory that are numbered by w & 3; the two warps of a quarter take the groups of 16
        // channels in turn.
        const int quarter = warp & 3, turn = (warp - 2) >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        OutT* out = (OutT*)p.out;
        wait_for_previous_kernel();
        let_next_kernel_start();
        int half = 0;
        uint32_t sums_parity = 0;                                 // one bit for each half
        for (int item = first; item < items; item += step) {
            int row0, expert, channel;
            place(item, row0, expert, channel);
            const int rows = listed ? min(p.lists.tile_rows, p.lists.offsets[expert + 1] - row0) : p.rows - row0;
            const int within = side * 128 + quarter * 32 + lane;
            const bool mine = within < rows && quarter * 32 + lane < p.x_box;
            const bool any = side * 128 + quarter * 32 < rows && quarter * 32 < p.x_box;
            const int row = row0 + within;
            const float x_scale = mine ? p.x_scale[row] : 0.f;
            const float* w_scale = p.w_scale + (size_t)expert * PARTS * p.FP + channel;
            const int channels = min(p.n, p.F - channel);
            if (!__all_sync(0xffffffffu, bar_wait(&sums_bar[half], (sums_parity >> half) & 1, failed))) { if (lane == 0) atomicExch(p.status, 125); break; }
            sums_parity ^= 1u << half;
            fence_after_sync();
            if (any) {
                const uint32_t sums = lanes + half * p.columns;
                OutT* dst = out + (size_t)row * p.F + channel;
                uint32_t acc[2][PARTS][16];
                int c = 16 * turn;
                if (c < channels) {
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) tmem_ld16(sums + q * p.n + c, acc[0][q]);
                }
#pragma unroll 1
                for (; c < channels; c += 64) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int c0 = c + 32 * h;
                        if (c0 >= channels) break;
                        float scale[PARTS][16];
#pragma unroll
                        for (int q = 0; q < PARTS; ++q)
#pragma unroll
                            for (int i = 0; i < 16; i += 4) {
                                const float4 v = __ldg(reinterpret_cast<const float4*>(w_scale + (size_t)q * p.FP + c0 + i));
                                scale[q][i] = v.x; scale[q][i + 1] = v.y; scale[q][i + 2] = v.z; scale[q][i + 3] = v.w;
                            }
                        tmem_wait_ld();
                        if (c0 + 32 < channels) {
#pragma unroll
                            for (int q = 0; q < PARTS; ++q) tmem_ld16(sums + q * p.n + c0 + 32, acc[h ^ 1][q]);
                        }
                        float v[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            v[i] = (float)(int)acc[h][0][i] * x_scale * scale[0][i];
                            if (PARTS == 2) v[i] = gated(v[i], (float)(int)acc[h][PARTS - 1][i] * x_scale * scale[PARTS - 1][i], p.gate, p.limit);
                        }
                        if (mine) store16(dst + c0, v, channels - c0, p.out_align);
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

static bool map_codes(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint32_t box_rows) {
    EncodeFn fn = encoder();
    if (!fn) return false;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {cols};
    cuuint32_t box[2] = {FRB_8BIT_KBLOCK, box_rows};
    cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Shape { int ctas, n; };

// Tokens that a block copies at a time: 128, or as many as a tile has where that is less.
static int tokens_box(const Product& p, int ctas) {
    const int tile = p.lists.tile_expert ? p.lists.tile_rows : p.rows;
    return ctas == 2 || tile >= 128 ? 128 : up_to(tile, 8);
}

// The form of a tile: the one whose last block is done first.  A block's k-block takes the tensor core 2 clocks a column and brings
// (tokens + its share of the weights' rows) * 128 bytes at about 50 bytes a clock and SM; a tile costs about 500 clocks besides.
static Shape choose(const Product& p, int sms) {
    const int k_blocks = up_to(p.K, FRB_8BIT_KBLOCK) / FRB_8BIT_KBLOCK;
    Shape best = {1, 32};
    double best_cost = 1e300;
    for (int ctas = 1; ctas <= 2; ++ctas) {
        const int tile_rows = p.lists.tile_expert ? p.lists.tile_rows : p.rows;
        if (p.lists.tile_expert ? (tile_rows > 128) != (ctas == 2) : ctas == 2 && p.rows <= 128) continue;
        const long long row_tiles = p.lists.tile_expert ? p.lists.max_tiles : (p.rows + 128 * ctas - 1) / (128 * ctas);
        const int x_box = tokens_box(p, ctas);
        for (int n = 16 * ctas; n * p.parts <= 256; n += 16 * ctas) {
            if (p.parts == 2 && ctas == 1 && n % 16) continue;
            const int columns = n * p.parts;
            const long long items = row_tiles * ((p.F + n - 1) / n), workers = sms / ctas;
            const double feed = (x_box + columns / ctas) * 128 / 50.0, math = 2.0 * columns;
            const double cost = (double)((items + workers - 1) / workers) * (k_blocks * (feed > math ? feed : math) + 500.0) + 8.0 * columns;
            if (cost < best_cost) { best_cost = cost; best = {ctas, n}; }
            if (n - 16 * ctas >= p.F) break;
        }
    }
    return best;
}

int product(const Product& q, cudaStream_t stream) {
    if (q.rows == 0 || (q.lists.tile_expert && q.lists.max_tiles == 0)) return 0;
    const int KP = up_to(q.K, FRB_8BIT_KBLOCK), FP = up_to(q.F, FRB_8BIT_ROWS);
    FRB_CHECK_ARG(q.K >= 1 && q.K <= FRB_8BIT_MOST_INNER, "product in 8 bits: an inner size of %d is outside 1..%d", q.K, FRB_8BIT_MOST_INNER);
    FRB_CHECK_ARG(q.F >= 1 && q.experts >= 1 && (q.parts == 1 || q.parts == 2), "product in 8 bits: %d experts of %d x %d channels", q.experts, q.parts, q.F);
    FRB_CHECK_ARG((((uintptr_t)q.w | (uintptr_t)q.x | (uintptr_t)q.w_scale) & 15) == 0, "product in 8 bits: codes and scales start on 16 bytes");
    FRB_CHECK_ARG(!q.lists.tile_expert || (q.lists.tile_rows >= 1 && q.lists.tile_rows <= 128) || q.lists.tile_rows == 256,
                  "product in 8 bits: tiles of %d rows (at most 128, or 256)", q.lists.tile_rows);
    const uint64_t w_rows = (uint64_t)q.experts * q.parts * FP;
    FRB_CHECK_ARG(w_rows < (1ull << 31) - 512, "product in 8 bits: %d experts of %d channels exceed a tensor map's rows", q.experts, q.F);
    const int sms = frb_sm_count();
    const Shape shape = choose(q, sms);
    const int ctas = shape.ctas;
    Params p;
    p.lists = q.lists; p.w_scale = q.w_scale; p.x_scale = q.x_scale; p.out = q.out; p.status = q.status;
    p.rows = q.rows; p.F = q.F; p.FP = FP; p.k_blocks = KP / FRB_8BIT_KBLOCK; p.gate = q.gate; p.limit = q.limit;
    p.n = shape.n;
    p.columns = p.n * q.parts;
    p.x_box = tokens_box(q, ctas);
    p.n_box = p.columns / ctas;
    const int two = 2 * p.columns;
    p.tmem_columns = two <= 32 ? 32 : two <= 64 ? 64 : two <= 128 ? 128 : two <= 256 ? 256 : 512;
    const int block_bytes = (p.x_box + p.n_box) * 128;
    // the A operand of an MMA is 128 rows, whatever was copied: the last stage's has to end inside the block's shared memory
    const int beyond = p.x_box < 128 ? 128 * 128 : 0;
    p.per_stage = 1;
    while (p.per_stage < 8 && p.per_stage * 2 * block_bytes <= 24 * 1024 && p.per_stage * 2 <= p.k_blocks) p.per_stage *= 2;
    p.stages = (P8_SMEM - 1024 - beyond) / (block_bytes * p.per_stage);
    if (p.stages > P8_MAX_STAGES) p.stages = P8_MAX_STAGES;
    p.row_tiles = (q.rows + 128 * ctas - 1) / (128 * ctas);
    p.channel_tiles = (q.F + p.n - 1) / p.n;
    const long long most = (long long)(q.lists.tile_expert ? q.lists.max_tiles : p.row_tiles) * p.channel_tiles;
    FRB_CHECK_ARG(most < (1ll << 31) - 4096, "product in 8 bits: %d rows of %d channels exceed the count of tiles", q.rows, q.F);
    const int row_bytes = q.F * (q.out_type == FRB_F32 ? 4 : 2);
    p.out_align = row_bytes % 32 == 0 && ((uintptr_t)q.out & 31) == 0 ? 2 : row_bytes % 16 == 0 && ((uintptr_t)q.out & 15) == 0 ? 1 : 0;
    CUtensorMap map_x, map_w;
    const uint32_t w_box = q.parts == 2 && ctas == 1 ? p.n : p.n_box;
    FRB_CHECK_ARG(map_codes(&map_x, q.x, q.rows, KP, p.x_box) && map_codes(&map_w, q.w, w_rows, KP, w_box),
                  "product in 8 bits: cuTensorMapEncodeTiled failed or is not available");
    const size_t smem = (size_t)p.stages * p.per_stage * block_bytes + beyond + 1024;
    const long long workers = sms / ctas;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)((most < workers ? most : workers) * ctas));
    config.blockDim = dim3(P8_THREADS);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = (unsigned)ctas;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
#define LAUNCH(CTAS, PARTS, OutT)                                                                                                     \
    do {                                                                                                                              \
        cudaFuncSetAttribute(product_8bit_kernel<CTAS, PARTS, OutT>, cudaFuncAttributeMaxDynamicSharedMemorySize, P8_SMEM);            \
        cudaLaunchKernelEx(&config, product_8bit_kernel<CTAS, PARTS, OutT>, map_x, map_w, p);                                         \
    } while (0)
    FRB_DISPATCH_DTYPE(q.out_type, OutT, {
        if (ctas == 2) { if (q.parts == 2) LAUNCH(2, 2, OutT); else LAUNCH(2, 1, OutT); }
        else { if (q.parts == 2) LAUNCH(1, 2, OutT); else LAUNCH(1, 1, OutT); }
    });
#undef LAUNCH
    FRB_RETURN_LAUNCH("product_8bit");
}

}  // namespace frb_products8
