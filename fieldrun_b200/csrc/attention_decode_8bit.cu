// One-token attention over a cache of 8-bit pages (cache_8bit.cuh), queries and outputs in bfloat16.
//
// For query head h over the keys j that its token may see (src/minimax.rs:270-281; the reference's form over 8-bit rows :317-347):
//     s_j = scale * ks_j * (q . kc_j),   out = sum_j exp(s_j - max) * vs_j * vc_j / sum_j exp(s_j - max),
// kc and vc the codes of key and value j, ks and vs their scales; with a cap, slopes, a sink or two maps as attention_decode_tma.
//
// What bounds it is the cache's bytes, dim + vdim + 8 a key and head.  They are half of the bfloat16 cache's, so everything a warp does
// with a key has to take half the time: the products are laid out with the keys as the rows of an MMA (S^T = K Q^T and O^T = V^T P^T,
// m16n8k16), where up to eight query heads of a key head fill the columns; with the heads as rows half of every MMA, of the
// accumulators and of the exponentials would belong to rows that do not exist.  Codes become float16 in registers, which is exact for
// both types; the queries are brought to float16 by a power of two per head (exact down to 2^-29 of a head's largest entry); a
// key's scale multiplies its scores, a value's scale its weight.
//
// A block takes a run of pages of one key head of one sequence, its warps the pages in turn.  A warp asks for its own pages by TMA
// (keys, then values, each announced on an mbarrier of the warp's own), the next page's keys as soon as the present page's scores are
// done and its values as soon as they are multiplied, so that a warp waits for nothing but its own copies; the page's number
// comes a page ahead.  The warps' results are combined through shared memory and written as one partial result; a second kernel
// joins the partial results in order.
//
// Weights: p_j = 2^(s_j - m) with m a running maximum that follows a page's only beyond a margin.  The weight that multiplies codes is
// w_j = p_j vs_j, rounded to float16 after division by a unit U per head, a power of two that follows the largest w seen: w / U is at most
// 2^15, and full precision (2^-11) reaches down to 2^-22 of the largest.  The sum of the p_j stays in float32.
//
// Which key a row of the score tile stands for, and which dimension a row of the output tile, is free; both are chosen so that the
// lanes of a quarter warp read shared memory from different banks under the copies' swizzle (key_of_row, below).
//
// Every wait on an mbarrier gives up after about a second and sets `status`; the block then waits (with the same limit) for the copies
// that are in flight and returns.
#include "cache_8bit.cuh"
#include "tma.cuh"

#define D8_WARPS 4
#define D8_THREADS (32 * D8_WARPS)
#define D8_CHUNK_PAGES 4               // a chunk is 256 keys
#define D8_RAISE 8.0f                  // the running maximum follows a page's maximum only beyond this margin (in units of log2)
#define D8_STATUS_WAIT 7               // a wait gave up
#define D8_STATUS_TOO_LONG 8           // a sequence has more keys than the launch was sized for

using namespace frb_tma;
using namespace frb_8bit;

struct Decode8Params {
    const bf16* q;             // [B, nh, HD]
    const float* k_scales;     // [pages, nkv, 64]
    const float* v_scales;     // [pages, v_heads, 64]
    const int* page_table;     // [slots, max_pages]
    const int* seq_pos;        // [B] position of the sequence's token; negative: the sequence has none, its output is zero
    const int* seq_slot;       // [B]
    float* part_o;             // [B, nh, parts, VD]
    float* part_ml;            // [B, nh, parts, 2]
    bf16* out;                 // [B, nh * VD], or with two maps per head [B, nh / 2 * VD]
    const float* slopes;       // as in DecodeAttnParams, like all below
    const float* sinks;
    const float* lam;
    int* status;
    float scale, softcap, diff_eps, diff_factor;
    int window, chunk, keep_first, max_pages, num_slots, num_pages, num_heads, num_kv_heads, v_heads;
    int parts, pages_per_block, head_tiles, early;
};

// The position that the kernels work with: none (-1) for a slot that does not exist.
__device__ __forceinline__ int held_position(const Decode8Params& p, int b) {
    const int slot = p.seq_slot[b];
    return slot >= 0 && slot < p.num_slots ? min(p.seq_pos[b], p.max_pages * FRB_PAGE - 1) : -1;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ float exp2_of(float x) {                 // 2^x by the special-function unit; below 2^-126: 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// e with 2^e <= x < 2^(e + 1), for normal x; 128 for infinity and NaN
__device__ __forceinline__ int exponent_of(float x) { return (int)((__float_as_uint(x) >> 23) & 0xffu) - 127; }

// The key, among eight neighbouring ones, that row r of eight rows of a score tile stands for.  Where a lane of a quarter warp reads 16 bytes
// of a value row of 128 bytes, the eight lanes read four rows (r = 2 t) and two neighbouring chunks of each; the copies put
// chunk c of row k at c ^ (k & 7), so the rows have to differ in bits 1 and 2; for a key row of 128 bytes they read two rows (r = 2 q,
// 2 q + 1), which have to differ in bit 2, and for one of 64 bytes, where two rows lie beside each other, in bit 0.  Value rows of
// 64 bytes are read eight bytes a lane, sixteen lanes at a time (four rows, half of each): the rows have to differ in bits 0 and 2.
template <int VD>
__device__ __forceinline__ int key_of_row(int r) {
    const int t = r >> 1, e = r & 1;
    return VD == 64 ? (((t & 1) ^ e) | (e << 1) | ((t >> 1) << 2)) : (((2 * t) ^ (4 * e)) + e);
}

// Byte offset of the 16-byte chunk c of row r in a tile that was copied with the swizzle of its row size.
template <int ROW>
__device__ __forceinline__ int chunk_at(int r, int c) {
    if (ROW == 128) c ^= r & 7;
    else if (ROW == 64) c ^= (r >> 1) & 3;
    else if (ROW == 32) c ^= (r >> 2) & 1;
    return r * ROW + 16 * c;
}

template <int BYTES> struct Words { uint32_t w[BYTES / 4]; };

// BYTES bytes that begin at byte `at` of row r.
template <int ROW, int BYTES>
__device__ __forceinline__ Words<BYTES> row_words(const uint8_t* tile, int r, int at) {
    Words<BYTES> v;
    if (BYTES == 16) {
        const uint4 x = *reinterpret_cast<const uint4*>(tile + chunk_at<ROW>(r, at >> 4));
        v.w[0] = x.x; v.w[1] = x.y; v.w[2] = x.z; v.w[3] = x.w;
    } else if (BYTES == 8) {
        const uint2 x = *reinterpret_cast<const uint2*>(tile + chunk_at<ROW>(r, at >> 4) + (at & 8));
        v.w[0] = x.x; v.w[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i)
            v.w[i] = *reinterpret_cast<const uint32_t*>(tile + chunk_at<ROW>(r, (at + 4 * i) >> 4) + ((at + 4 * i) & 12));
    }
    return v;
}

// Four codes of a key as two float16 pairs (entries 0 1 | 2 3 for e4m3, 0 2 | 1 3 for int8: the queries are paired alike).
template <int CODES>
__device__ __forceinline__ void key_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (CODES == FRB_E4M3) halves_of_e4m3(w, lo, hi);
    else { lo = half_of_int8(w); hi = half_of_int8(w >> 8); }
}

// Entries 2 n and 2 n + 1 (n = 0, 1) of four codes of two keys: entry 2 n of both as `even`, entry 2 n + 1 as `odd`.
template <int CODES>
__device__ __forceinline__ void value_halves(uint32_t first, uint32_t second, int n, uint32_t& even, uint32_t& odd) {
    if (CODES == FRB_E4M3) {
        halves_of_e4m3(__byte_perm(first, second, n == 0 ? 0x5140 : 0x7362), even, odd);
    } else {
        even = half_of_int8(__byte_perm(first, second, n == 0 ? 0x0400 : 0x0602));       // bytes 0 and 2 count
        odd = half_of_int8(__byte_perm(first, second, n == 0 ? 0x0501 : 0x0703));
    }
}

__device__ __forceinline__ void load_row_of_scales(void* dst, const float* src, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_addr(dst)), "l"(src), "r"(4 * FRB_PAGE), "r"(smem_addr(bar)) : "memory");
}

// HD, VD: entries of a key and of a value head.  NT: query heads of a key head in tiles of eight (1 or 2); a block takes NT tiles.
template <int HD, int VD, int NT, int CODES>
__global__ void __launch_bounds__(D8_THREADS, NT == 1 ? 3 : 2)
attention_decode_8bit_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Decode8Params p) {
    // as attention_decode_tma: the copies of every page but the sequence's last go out before the kernel before this one has ended
    let_next_kernel_start();
    constexpr int K_TILE = FRB_PAGE * HD, V_TILE = FRB_PAGE * VD, SCALES = 4 * FRB_PAGE;
    constexpr int KU = HD % 64 == 0 ? 16 : 8, K_STEPS = HD / (4 * KU), K_WORDS = KU / 4;     // a lane's bytes of a key at a time
    constexpr int VB = VD / 8, MT = VD / 16;                                                // a lane's bytes of a value; output tiles
    constexpr int O_STRIDE = VD + 4;
    static_assert(NT * 8 * O_STRIDE * 4 <= K_TILE + V_TILE, "a warp's partial result fits into its pages");
    extern __shared__ uint8_t dynamic[];
    __shared__ uint64_t full_k[D8_WARPS], full_v[D8_WARPS];
    __shared__ float sm_m[D8_WARPS][8 * NT], sm_l[D8_WARPS][8 * NT];
    __shared__ int failed;
    uint8_t* tiles = reinterpret_cast<uint8_t*>(((uintptr_t)dynamic + 1023) & ~(uintptr_t)1023);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint8_t* k_tile = tiles + (size_t)warp * (K_TILE + V_TILE);
    uint8_t* v_tile = k_tile + K_TILE;
    float* k_scale = reinterpret_cast<float*>(tiles + (size_t)D8_WARPS * (K_TILE + V_TILE) + (size_t)warp * 2 * SCALES);
    float* v_scale = k_scale + FRB_PAGE;

    const int part = blockIdx.x, kvh = blockIdx.y / p.head_tiles, tile = blockIdx.y - kvh * p.head_tiles, b = blockIdx.z;
    const int group = p.num_heads / p.num_kv_heads;
    const int first_head = kvh * group + tile * 8 * NT, heads = min(8 * NT, group - tile * 8 * NT);
    const int hi_key = held_position(p, b), lo_key = first_visible_key(max(hi_key, 0), p.window, p.chunk);
    // the pages of this block that hold a key the token may see: those of the first tokens that stay visible, then the window's
    const int begin_page = part * p.pages_per_block, end_page = min((part + 1) * p.pages_per_block, hi_key < 0 ? 0 : hi_key / FRB_PAGE + 1);
    const int first_page = max(begin_page, lo_key / FRB_PAGE);
    const int kept = max(0, min(end_page, kept_runs(p.keep_first, FRB_PAGE, lo_key / FRB_PAGE)) - begin_page);
    const int num_pages = kept + max(0, end_page - first_page);
    if (num_pages <= 0) return;                   // the join skips these blocks
    const auto number_of = [&](int n) { return n < kept ? begin_page + n : first_page + n - kept; };
    const int* table = p.page_table + (size_t)p.seq_slot[b] * p.max_pages;
    // the store's page of the run's page n; -1 behind the run's end and for one that the table does not have
    const auto page_of = [&](int n) {
        if (n >= num_pages) return -1;
        const int page = table[number_of(n)];
        return page < p.num_pages ? page : -1;
    };
    const int vh = kvh / (p.num_kv_heads / p.v_heads);

    if (threadIdx.x == 0) {
        for (int w = 0; w < D8_WARPS; ++w) { bar_init(&full_k[w], 1); bar_init(&full_v[w], 1); }
        failed = 0;
        bar_init_fence();
    }
    __syncthreads();

    const auto ask_keys = [&](int page) {
        bar_expect(&full_k[warp], K_TILE + SCALES);
        load_2d(k_tile, &map_k, 0, (page * p.num_kv_heads + kvh) * FRB_PAGE, &full_k[warp]);
        load_row_of_scales(k_scale, p.k_scales + ((size_t)page * p.num_kv_heads + kvh) * FRB_PAGE, &full_k[warp]);
    };
    const auto ask_values = [&](int page) {
        bar_expect(&full_v[warp], V_TILE + SCALES);
        load_2d(v_tile, &map_v, 0, (page * p.v_heads + vh) * FRB_PAGE, &full_v[warp]);
        load_row_of_scales(v_scale, p.v_scales + ((size_t)page * p.v_heads + vh) * FRB_PAGE, &full_v[warp]);
    };

    // Copies in flight at any time: the keys and the values of page `page`.  The run's page n is this warp's for n = warp, warp +
    // D8_WARPS, ...; pages that the table does not have are passed over.
    int n = warp, page = -1;
    const auto next_page = [&](int from) {                  // the warp's first page from the run's page `from` on
        n = from;
        for (page = -1; n < num_pages && page < 0; n += page < 0 ? D8_WARPS : 0) page = page_of(n);
    };
    const int newest = kept + hi_key / FRB_PAGE - first_page;       // the page that the kernel before this one writes to
    bool waited = !p.early;
    if (waited) wait_for_previous_kernel();
    next_page(warp);
    if (page >= 0 && (waited || n != newest) && lane == 0) { ask_keys(page); ask_values(page); }
    if (!waited) {
        wait_for_previous_kernel();
        if (page >= 0 && n == newest && lane == 0) { ask_keys(page); ask_values(page); }
    }

    // the queries: head g of a tile, entries as the keys' words have them
    uint32_t q[NT][K_STEPS * K_WORDS][2];
    float s_scale[NT][2], slope2[NT][2];                     // heads 2 t and 2 t + 1: scores to units of log2, or for a cap to units of the cap
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const bf16* row = p.q + ((size_t)b * p.num_heads + first_head + 8 * j + g) * HD;
        float x[K_STEPS * K_WORDS][4];
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < K_STEPS; ++s)
#pragma unroll
            for (int w = 0; w < K_WORDS; ++w) {
                const float4 v = 8 * j + g < heads ? load4<bf16>(row + (4 * s + t) * KU + 4 * w) : make_float4(0.f, 0.f, 0.f, 0.f);
                float (&to)[4] = x[s * K_WORDS + w];
                to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(to[e]));
            }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = max(exponent_of(top), -100);           // |q| 2^(14 - e) < 2^15
        const float factor = power_of_two(14 - min(e, 127));
        const float unit = power_of_two(min(e, 127) - 14) * (p.softcap > 0.f ? p.scale / p.softcap : p.scale * 1.4426950408889634f);
#pragma unroll
        for (int i = 0; i < K_STEPS * K_WORDS; ++i) {
            const bool plain = CODES == FRB_E4M3;
            q[j][i][0] = pack_f16(x[i][0] * factor, x[i][plain ? 1 : 2] * factor);
            q[j][i][1] = pack_f16(x[i][plain ? 2 : 1] * factor, x[i][3] * factor);
        }
        s_scale[j][0] = __shfl_sync(0xffffffffu, unit, 8 * t);
        s_scale[j][1] = __shfl_sync(0xffffffffu, unit, 8 * t + 4);
#pragma unroll
        for (int c = 0; c < 2; ++c)
            slope2[j][c] = p.slopes && 8 * j + 2 * t + c < heads ? p.slopes[first_head + 8 * j + 2 * t + c] * 1.4426950408889634f : 0.f;
    }
    const float cap2 = p.softcap > 0.f ? p.softcap * 1.4426950408889634f : 0.f;

    float row_max[NT][2], row_sum[NT][2], unit[NT][2], inverse[NT][2];
    float o[NT][MT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int c = 0; c < 2; ++c) { row_max[j][c] = -INFINITY; row_sum[j][c] = 0.f; unit[j][c] = 0.f; inverse[j][c] = 0.f; }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][i][e] = 0.f;
    }

    uint32_t k_parity = 0, v_parity = 0;
    bool keys_out = page >= 0, values_out = page >= 0;      // a copy is in flight
    bool cleared = false;                                   // this warp wrote into its tiles
    while (page >= 0) {
        const int key_base = number_of(n) * FRB_PAGE;
        const bool edge = key_base < lo_key || key_base + FRB_PAGE - 1 > hi_key;
        next_page(n + D8_WARPS);                            // the next one's number is there when its copy is asked for
        if (!__all_sync(0xffffffffu, bar_wait(&full_k[warp], k_parity, &failed))) break;
        k_parity ^= 1;
        keys_out = false;
        float s[NT][4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {                       // sixteen keys: rows g and g + 8 of the tile
            const int k0 = 16 * i + key_of_row<VD>(g), k1 = k0 + 8;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][i][e] = 0.f;
#pragma unroll
            for (int step = 0; step < K_STEPS; ++step) {
                const Words<KU> a = row_words<HD, KU>(k_tile, k0, (4 * step + t) * KU), c = row_words<HD, KU>(k_tile, k1, (4 * step + t) * KU);
#pragma unroll
                for (int w = 0; w < K_WORDS; ++w) {
                    uint32_t a0, a1, a2, a3;
                    key_halves<CODES>(a.w[w], a0, a2);
                    key_halves<CODES>(c.w[w], a1, a3);
#pragma unroll
                    for (int j = 0; j < NT; ++j) mma_f16(s[j][i], a0, a1, a2, a3, q[j][step * K_WORDS + w][0], q[j][step * K_WORDS + w][1]);
                }
            }
            const float ks0 = k_scale[k0], ks1 = k_scale[k1];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float scaled = s[j][i][e] * (s_scale[j][e & 1] * (e < 2 ? ks0 : ks1));
                    // (the cap's minimum would turn NaN into a number)
                    const float score = cap2 > 0.f && scaled == scaled ? capped_score2(scaled, 1.f, cap2) : scaled;
                    s[j][i][e] = fmaf(slope2[j][e & 1], (float)(key_base + (e < 2 ? k0 : k1) - hi_key), score);
                }
        }
        __syncwarp();
        if (page >= 0 && lane == 0) ask_keys(page);          // this page's keys are no longer needed
        keys_out = page >= 0;
        // only the pages at the window's edge, behind the first tokens and of the token itself hold keys it may not see
        if (edge) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!key_visible(key_base + 16 * i + key_of_row<VD>(g) + (e < 2 ? 0 : 8), lo_key, hi_key, p.keep_first))
                            s[j][i][e] = -INFINITY;
        }
        float page_max[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float top = s[j][0][c];
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(s[j][i][c], s[j][i][c + 2]));
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                page_max[j][c] = top;
            }
        float corr[NT][2];
        bool grew = false;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                corr[j][c] = 1.f;
                if (page_max[j][c] > row_max[j][c] + D8_RAISE) {      // also on the warp's first page
                    corr[j][c] = exp2_of(row_max[j][c] - page_max[j][c]);
                    row_max[j][c] = page_max[j][c];
                    grew = true;
                }
            }
        if (!__all_sync(0xffffffffu, bar_wait(&full_v[warp], v_parity, &failed))) break;
        v_parity ^= 1;
        values_out = false;
        if (edge) {
            // whatever lies in the places of keys that the token may not see (their weight is zero, but zero times NaN is not)
            for (int k = 0; k < FRB_PAGE; ++k)
                if (!key_visible(key_base + k, lo_key, hi_key, p.keep_first)) {
                    if (4 * lane < VD) *reinterpret_cast<uint32_t*>(v_tile + k * VD + 4 * lane) = 0u;
                    if (lane == 0) v_scale[k] = 0.f;
                }
            cleared = true;
            __syncwarp();
        }
        float top_w[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) { row_sum[j][c] *= corr[j][c]; top_w[j][c] = 0.f; }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k0 = 16 * i + key_of_row<VD>(g);
            const float vs0 = v_scale[k0], vs1 = v_scale[k0 + 8];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float weight = exp2_of(s[j][i][e] - row_max[j][e & 1]);
                    row_sum[j][e & 1] += weight;
                    s[j][i][e] = weight * (e < 2 ? vs0 : vs1);
                    top_w[j][e & 1] = fmaxf(top_w[j][e & 1], s[j][i][e]);
                }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top_w[j][c] = fmaxf(top_w[j][c], __shfl_xor_sync(0xffffffffu, top_w[j][c], d));
                if (top_w[j][c] * inverse[j][c] > 32768.f || (unit[j][c] == 0.f && top_w[j][c] > 0.f)) {
                    const int e = min(max(exponent_of(top_w[j][c]) - 7, -119), 119);
                    corr[j][c] *= unit[j][c] * power_of_two(-e);
                    unit[j][c] = power_of_two(e);
                    inverse[j][c] = power_of_two(-e);
                    grew = true;
                }
            }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    o[j][i][0] *= corr[j][0]; o[j][i][1] *= corr[j][1];
                    o[j][i][2] *= corr[j][0]; o[j][i][3] *= corr[j][1];
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t b0[NT], b1[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {                  // rows g of eight keys, columns 2 t, 2 t + 1 -> keys 2 t, 2 t + 1 of head g
                b0[j] = transposed_8x8(pack_f16(s[j][i][0] * inverse[j][0], s[j][i][1] * inverse[j][1]));
                b1[j] = transposed_8x8(pack_f16(s[j][i][2] * inverse[j][0], s[j][i][3] * inverse[j][1]));
            }
            const int ka = 16 * i + key_of_row<VD>(2 * t), kb = 16 * i + key_of_row<VD>(2 * t + 1);
            const Words<VB> va = row_words<VD, VB>(v_tile, ka, VB * g), vb = row_words<VD, VB>(v_tile, kb, VB * g);
            const Words<VB> vc = row_words<VD, VB>(v_tile, ka + 8, VB * g), vd = row_words<VD, VB>(v_tile, kb + 8, VB * g);
#pragma unroll
            for (int m = 0; m < MT; ++m) {                  // rows g and g + 8: dimensions VB g + 2 m and + 1
                uint32_t a0, a1, a2, a3;
                value_halves<CODES>(va.w[m >> 1], vb.w[m >> 1], m & 1, a0, a1);
                value_halves<CODES>(vc.w[m >> 1], vd.w[m >> 1], m & 1, a2, a3);
#pragma unroll
                for (int j = 0; j < NT; ++j) mma_f16(o[j][m], a0, a1, a2, a3, b0[j], b1[j]);
            }
        }
        if (cleared) {                                      // ordinary stores into the tile, before a copy writes there again
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            cleared = false;
        }
        __syncwarp();
        if (page >= 0 && lane == 0) ask_values(page);
        values_out = page >= 0;
    }
    // a warp that gave up leaves only when the copies that it asked for have landed (or a second limit has passed)
    if (keys_out || values_out) {
        int again = 0;
        if (keys_out) bar_wait(&full_k[warp], k_parity, &again);
        if (values_out) bar_wait(&full_v[warp], v_parity, &again);
        failed = 1;
    }
    __syncthreads();
    if (failed) {
        if (threadIdx.x == 0) *p.status = D8_STATUS_WAIT;
        return;
    }
    float* mine = reinterpret_cast<float*>(k_tile);          // [8 NT heads][O_STRIDE]
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) row_sum[j][c] += __shfl_xor_sync(0xffffffffu, row_sum[j][c], d);
            float* row = mine + (8 * j + 2 * t + c) * O_STRIDE;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                row[VB * g + 2 * m] = o[j][m][c] * unit[j][c];
                row[VB * g + 2 * m + 1] = o[j][m][c + 2] * unit[j][c];
            }
            if (g == 0) { sm_m[warp][8 * j + 2 * t + c] = row_max[j][c]; sm_l[warp][8 * j + 2 * t + c] = row_sum[j][c]; }
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < heads * VD; idx += D8_THREADS) {
        const int r = idx / VD, d = idx - r * VD;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < D8_WARPS; ++w) top = fmaxf(top, sm_m[w][r]);
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < D8_WARPS; ++w) {
            if (sm_l[w][r] != 0.f) {                        // a warp that had no page wrote zeros and no maximum
                const float f = exp2f(sm_m[w][r] - top);
                sum += sm_l[w][r] * f;
                acc += reinterpret_cast<const float*>(tiles + (size_t)w * (K_TILE + V_TILE))[r * O_STRIDE + d] * f;
            }
        }
        const size_t row = ((size_t)b * p.num_heads + first_head + r) * p.parts + part;
        p.part_o[row * VD + d] = acc;
        if (d == 0) { p.part_ml[row * 2] = top; p.part_ml[row * 2 + 1] = sum; }
    }
}

// Entry d of the joined output of one (sequence, head): partial results 0 .. kept - 1, then first .. last, in that order, eight at a
// time (all of their loads before the first use).  A partial result without a key (maximum -inf, sum 0) adds nothing; without any the
// output is zero, with a sink or not.
template <int VD>
__device__ __forceinline__ float joined_8bit(const float* __restrict__ part_ml, const float* __restrict__ part_o, size_t row0, int kept,
                                             int first, int last, int d, float sink2) {
    constexpr int AT_ONCE = 8;
    float top = -INFINITY, sum = 0.f, acc = 0.f;
    const int end = kept + last - first;
    for (int c0 = 0; c0 <= end; c0 += AT_ONCE) {
        float2 ml[AT_ONCE];
        float o[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int c = run_at(min(c0 + u, end), kept, first);
            ml[u] = *reinterpret_cast<const float2*>(part_ml + (row0 + c) * 2);
            o[u] = part_o[(row0 + c) * VD + d];
        }
        float group_top = top;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
            if (c0 + u <= end) group_top = fmaxf(group_top, ml[u].x);
        const float keep = sum == 0.f ? 0.f : exp2f(top - group_top);
        sum *= keep;
        acc *= keep;
        top = group_top;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
            if (c0 + u <= end && ml[u].y != 0.f) {
                const float f = exp2f(ml[u].x - top);
                sum += ml[u].y * f;
                acc += o[u] * f;
            }
    }
    if (sum == 0.f) return 0.f;
    if (sink2 > -INFINITY) {                              // a sink: a term of the denominator without a value
        const float top_all = fmaxf(top, sink2);
        const float keep = exp2f(top - top_all);
        sum = sum * keep + exp2f(sink2 - top_all);
        acc *= keep;
    }
    return acc / sum;
}

// grid (output head, sequence), a thread per value entry.
template <int VD>
__global__ void __launch_bounds__(VD) attention_decode_8bit_join_kernel(Decode8Params p) {
    after_previous_kernel();
    __shared__ float scratch[32];
    const int head = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
    const int pos = held_position(p, b), keys_per_part = p.pages_per_block * FRB_PAGE;
    const int heads = p.lam ? p.num_heads / 2 : p.num_heads;
    bf16* out = p.out + ((size_t)b * heads + head) * VD + d;
    if (pos < 0) { *out = __float2bfloat16_rn(0.f); return; }
    const int lo_key = first_visible_key(pos, p.window, p.chunk);
    const int last = min(pos / keys_per_part, p.parts - 1), first = min(lo_key / keys_per_part, last);
    const int kept = kept_runs(p.keep_first, keys_per_part, first);
    if (pos / keys_per_part >= p.parts && d == 0) atomicExch(p.status, D8_STATUS_TOO_LONG);   // keys were left out
    if (p.lam) {
        const int group = p.num_heads / p.num_kv_heads, g = head / group;
        const size_t row1 = ((size_t)b * p.num_heads + (size_t)(2 * g) * group + (head - g * group)) * p.parts;
        const size_t row2 = row1 + (size_t)group * p.parts;
        const float a1 = joined_8bit<VD>(p.part_ml, p.part_o, row1, kept, first, last, d, -INFINITY);
        const float a2 = joined_8bit<VD>(p.part_ml, p.part_o, row2, kept, first, last, d, -INFINITY);
        const float o = a1 - *p.lam * a2;
        const float ss = block_sum<VD>(o * o, scratch);
        *out = __float2bfloat16_rn(o / sqrtf(ss / (float)VD + p.diff_eps) * p.diff_factor);
        return;
    }
    *out = __float2bfloat16_rn(joined_8bit<VD>(p.part_ml, p.part_o, ((size_t)b * p.num_heads + head) * p.parts, kept, first, last, d,
                                               p.sinks ? p.sinks[head] * 1.4426950408889634f : -INFINITY));
}

// A map over rows of `row` one-byte codes, boxes of 64 rows with the swizzle of the row's size.
static bool map_code_rows(CUtensorMap* map, const void* base, uint64_t rows, int row) {
    EncodeFn fn = encoder();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)row, rows};
    cuuint64_t strides[1] = {(cuuint64_t)row};
    cuuint32_t box[2] = {(cuuint32_t)row, FRB_PAGE};
    cuuint32_t elem[2] = {1, 1};
    const CUtensorMapSwizzle swizzle = row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : row == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                       : row == 32 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_NONE;
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, int VD, int NT, int CODES>
static void launch_decode_8bit(const CUtensorMap& map_k, const CUtensorMap& map_v, const Decode8Params& p, dim3 grid, cudaStream_t stream) {
    const size_t smem = (size_t)D8_WARPS * (FRB_PAGE * (HD + VD) + 8 * FRB_PAGE) + 1024;
    auto kernel = attention_decode_8bit_kernel<HD, VD, NT, CODES>;
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    launch_dependent_resident(p.early ? (NT == 1 ? 3 : 2) : 1, kernel, grid, dim3(D8_THREADS), smem, stream, map_k, map_v, p);
}

// max_chunks: chunks of 256 keys of the longest sequence; part_o and part_ml hold ceil(max_chunks / chunks_per_block) partial results per
// (sequence, head).  num_pages: pages of the store.  status: one int on the device.
FRB_API int frb_attention_decode_8bit(const void* q, const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales,
                                      int codes, int num_pages, const int* page_table, int num_slots, int max_pages, const int* seq_pos,
                                      const int* seq_slot, float* part_o, float* part_ml, void* out, int num_seqs, int num_heads,
                                      int num_kv_heads, int v_heads, int head_dim, int v_dim, float scale, int window, int chunk,
                                      int keep_first, int max_chunks, int chunks_per_block, const float* slopes, const float* sinks,
                                      float softcap, const float* lam, float diff_eps, float diff_factor, int* status,
                                      cudaStream_t stream) {
    if (num_seqs == 0) return 0;
    FRB_CHECK_ARG(num_seqs > 0 && num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0 && v_heads > 0 && num_kv_heads % v_heads == 0,
                  "attention_decode_8bit: %d sequences, %d heads over %d key heads and %d value heads", num_seqs, num_heads, num_kv_heads, v_heads);
    FRB_CHECK_ARG(codes == FRB_E4M3 || codes == FRB_INT8, "attention_decode_8bit: codes of type %d", codes);
    FRB_CHECK_ARG(num_pages > 0 && num_slots > 0 && max_pages > 0 && max_pages < (1 << 25), "attention_decode_8bit: %d pages, %d slots of %d",
                  num_pages, num_slots, max_pages);
    FRB_CHECK_ARG((long long)num_pages * num_kv_heads * FRB_PAGE < (1ll << 31), "attention_decode_8bit: %d pages of %d heads exceed a tensor map's rows",
                  num_pages, num_kv_heads);
    FRB_CHECK_ARG(chunks_per_block >= 1 && max_chunks >= 1, "attention_decode_8bit: %d chunks, %d per block", max_chunks, chunks_per_block);
    FRB_CHECK_ARG(window >= 0 && chunk >= 0 && keep_first >= 0 && !(keep_first > 0 && chunk > 0),
                  "attention_decode_8bit: a window of %d, chunks of %d, %d first tokens", window, chunk, keep_first);
    FRB_CHECK_ARG(!lam || (num_kv_heads == 2 * v_heads && !sinks), "attention_decode_8bit: two maps per head need two key heads a value head and no sinks");
    const auto aligned = [](const void* ptr, uintptr_t bytes) { return ((uintptr_t)ptr & (bytes - 1)) == 0; };
    FRB_CHECK_ARG(aligned(q, 8) && aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(k_scales, 16) && aligned(v_scales, 16) && aligned(part_ml, 8),
                  "attention_decode_8bit: queries start on 8 bytes, codes and scales on 16");
    const int group = num_heads / num_kv_heads, per_block = group <= 8 ? 8 : 16, head_tiles = (group + per_block - 1) / per_block;
    FRB_CHECK_ARG(num_seqs <= 65535 && (long long)num_kv_heads * head_tiles <= 65535, "attention_decode_8bit: %d sequences of %d heads exceed the grid",
                  num_seqs, num_heads);
    Decode8Params p;
    p.q = (const bf16*)q; p.k_scales = k_scales; p.v_scales = v_scales; p.page_table = page_table; p.seq_pos = seq_pos; p.seq_slot = seq_slot;
    p.part_o = part_o; p.part_ml = part_ml; p.out = (bf16*)out; p.slopes = slopes; p.sinks = sinks; p.lam = lam; p.status = status;
    p.scale = scale; p.softcap = softcap > 0.f ? softcap : 0.f; p.diff_eps = diff_eps; p.diff_factor = diff_factor; p.window = window;
    p.chunk = chunk; p.keep_first = window > 0 ? keep_first : 0; p.max_pages = max_pages; p.num_slots = num_slots; p.num_pages = num_pages;
    p.num_heads = num_heads; p.num_kv_heads = num_kv_heads; p.v_heads = v_heads; p.parts = (max_chunks + chunks_per_block - 1) / chunks_per_block;
    p.pages_per_block = chunks_per_block * D8_CHUNK_PAGES; p.head_tiles = head_tiles;
    static const int early = [] { const char* v = getenv("FIELDRUN_B200_ATTENTION_EARLY"); return !(v && v[0] == '0'); }();
    p.early = early;
    CUtensorMap map_k, map_v;
    FRB_CHECK_ARG(map_code_rows(&map_k, k_codes, (uint64_t)num_pages * num_kv_heads * FRB_PAGE, head_dim) &&
                  map_code_rows(&map_v, v_codes, (uint64_t)num_pages * v_heads * FRB_PAGE, v_dim),
                  "attention_decode_8bit: head_dim %d with value heads of %d: cuTensorMapEncodeTiled failed or is not available", head_dim, v_dim);
    const dim3 grid(p.parts, num_kv_heads * head_tiles, num_seqs), join_grid(lam ? num_heads / 2 : num_heads, num_seqs);
#define FRB_LAUNCH_DECODE8(HD, VD)                                                                                                  \
    if (per_block == 8 && codes == FRB_E4M3) launch_decode_8bit<HD, VD, 1, FRB_E4M3>(map_k, map_v, p, grid, stream);                \
    else if (per_block == 8) launch_decode_8bit<HD, VD, 1, FRB_INT8>(map_k, map_v, p, grid, stream);                                \
    else if (codes == FRB_E4M3) launch_decode_8bit<HD, VD, 2, FRB_E4M3>(map_k, map_v, p, grid, stream);                             \
    else launch_decode_8bit<HD, VD, 2, FRB_INT8>(map_k, map_v, p, grid, stream);                                                    \
    launch_dependent(attention_decode_8bit_join_kernel<VD>, join_grid, dim3(VD), 0, stream, p)
    FRB_8BIT_SIZES("attention_decode_8bit", head_dim, v_dim, FRB_LAUNCH_DECODE8);
#undef FRB_LAUNCH_DECODE8
    FRB_RETURN_LAUNCH("attention_decode_8bit");
}
