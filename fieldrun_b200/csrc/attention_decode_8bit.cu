// One-token attention over a cache of 8-bit pages (cache_8bit.cuh), queries and outputs in bfloat16.
//
// For query head h over the keys j that its token may see (src/minimax.rs:270-281; the reference's form over 8-bit rows :317-347):
//     s_j = scale * ks_j * (q . kc_j),   out = sum_j exp(s_j - max) * vs_j * vc_j / sum_j exp(s_j - max),
// kc and vc the codes of key and value j, ks and vs their scales; with a cap, slopes, a sink or two maps as attention_decode_tma.
//
// What bounds it is the cache's bytes, dim + vdim + 8 a key and head.  They are half of the bfloat16 cache's, so everything a warp does
// with a key has to take half the time: the products are laid out with the keys as the rows of an MMA (S^T = K Q^T and O^T = V^T P^T,
// m16n8k16), where up to eight query heads of a key head fill the columns; with the heads as rows half of every MMA, of the
// accumulators and of the exponentials would belong to rows that do not exist.  A key's scale multiplies its scores, a value's its weight.
//
// Scores: codes of either type become float16 in registers, which is exact, and the queries are brought to float16 by a power of two per head
// (exact down to 2^-29 of a head's largest entry): what a score loses is lost in float32 sums.  (int8 codes multiplied as they are, by queries in two
// parts of 8 bits, take 55 us for 32 sequences of 4,096 keys where this takes 57, but round every query entry to 2^-16 of the head's largest: where
// that one meets keys of zero and is 1,000 times the others, outputs are off by 4 per cent.  The products of e4m3 codes are no instruction of
// their own for single warps: with them, and the queries in two e4m3 parts, the same sequences took 71 us, with float16 58.)
//
// Weights: p_j = 2^(s_j - m) with m a running maximum that follows a page's only beyond a margin.  The weight that multiplies codes is
// w_j = p_j vs_j, rounded to float16 after division by a unit U per head, a power of two that follows the largest w seen: w / U is at most
// 2^15, and full precision (2^-11) reaches down to 2^-22 of the largest so far.  U only grows: where the running maximum has risen since, the outputs
// shrink and U does not, so that beside an early value row 10^7 times the others these have fewer digits.  The sum of the p_j stays in float32.
//
// A page of 64 keys is one warp's work: its keys and values come by TMA into tiles of the warp's own, each announced on an mbarrier of
// the warp's own.  Which key a row of the score tile stands for, and which dimension a row of the output tile, is free; both are
// chosen so that the lanes of a quarter warp read shared memory from different banks under the copies' swizzle (key_of_row).
//
// Two kernels cut the work differently (the entry point chooses), a third joins the partial results in order:
// chunks: a block takes four pages of a key head, a page a warp, and combines the four through shared memory.  Where there are few pages
//   nothing is faster: every page is read at once.
// pieces: all pages that the step's tokens see, sequence by sequence and key head by key head, are one line that is cut into pieces of one
//   length, a warp's each, about as many as warps are resident.  A warp runs through its piece without waiting for any other: the
//   next page's keys are asked for as soon as the present page's scores are done and its values as soon as they are multiplied, also from
//   one key head or sequence to the next, where the warp leaves a partial result.  Sequences of unequal lengths need no more time than
//   their pages, and there is no last wave of a few blocks.  Where a head has room for too few partial results, cut between key heads only.
//
// Measured on a B200, 48 heads on 8 key heads of 128: 32 sequences of 4,096 keys 54 us (e4m3; 277 MB, 5.1 TB/s; 52 of them the pieces, issue slots 35 %
// busy, 9 to 10 warps an SM; pages of bfloat16 take 92 us), one of 131,072 keys 58 us (int8, issue slots 50 %
// busy), one of 2,048 keys 6.5 us.
//
// Every wait on an mbarrier gives up after about a second and sets `status`; the warps then wait (with the same limit) for the copies
// that are in flight and return.
#include "cache_8bit.cuh"
#include "step_rows.h"
#include "tma.cuh"

#define D8_WARPS 4
#define D8_THREADS (32 * D8_WARPS)
// Blocks that an SM holds: their pages fill its shared memory (heads of 128: 203 of 227 KB) or their registers its file (128 a thread
// for the smaller heads, 168).
#define D8_RESIDENT(HD, VD, NT) ((NT) == 2 ? 2 : (HD) + (VD) <= 128 ? 4 : 3)
#define D8_CHUNK_PAGES 4               // a chunk is 256 keys
#define D8_LEAD 2                      // pages that a run costs as much time as, beside its own (64 ragged sequences in windows: 0 59 us, 2 47 us)
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
    float* part_o;             // [B, nh, max_chunks, VD]
    float* part_ml;            // [B, nh, max_chunks, 2]
    bf16* out;                 // [B, nh * VD], or with two maps per head [B, nh / 2 * VD]
    const float* slopes;       // null, or one slope per query head: key j's score is lowered by slope * (position - j)
    const float* sinks;        // null, or one number per query head whose exponential joins the softmax's denominator
    const float* lam;          // not null: two maps per head; query heads lie as [value head, map, query head of the group]
    int* status;
    float scale, softcap, diff_eps, diff_factor;
    int window, chunk, keep_first, max_pages, num_slots, num_pages, num_heads, num_kv_heads, v_heads, num_seqs;
    int max_chunks;            // partial results that there is room for per (sequence, head); a sequence has at most four times as many pages
    int head_tiles;            // tiles of query heads per key head
    int pieces;                // warps that the line of pages is cut for; 0: chunks
    int whole;                 // a key head's pages are one piece's, since there is no room for partial results
    int early;                 // copies go out before the kernel before this one has ended (0: FIELDRUN_B200_ATTENTION_EARLY=0)
};

// The pages that hold a key which a sequence's token may see: those of the first tokens that stay visible, then the window's.
struct Sight {
    int lo_key, hi_key, kept, first_page, count;
    bool cut;                                           // there are more, which the launch has no room for
    __device__ __forceinline__ int number(int n) const { return n < kept ? n : first_page + n - kept; }     // the n-th one's place in the sequence
};

// of a token at `position` of `slot`; a slot that does not exist has none
__device__ __forceinline__ Sight sight_from(const Decode8Params& p, int slot, int position) {
    Sight s;
    s.hi_key = slot >= 0 && slot < p.num_slots ? min(position, p.max_pages * FRB_PAGE - 1) : -1;
    s.lo_key = first_visible_key(max(s.hi_key, 0), p.window, p.chunk);
    s.first_page = s.lo_key / FRB_PAGE;
    s.kept = kept_runs(p.keep_first, FRB_PAGE, s.first_page);
    const int pages = s.hi_key < 0 ? 0 : s.kept + s.hi_key / FRB_PAGE + 1 - s.first_page;
    s.cut = pages > D8_CHUNK_PAGES * p.max_chunks;
    s.count = s.cut ? D8_CHUNK_PAGES * p.max_chunks : pages;
    return s;
}

__device__ __forceinline__ Sight sight_of(const Decode8Params& p, int b) { return sight_from(p, p.seq_slot[b], p.seq_pos[b]); }

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
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

// Four codes of a key as two float16 pairs, and four query entries as the pairs that they are multiplied with.  e4m3: entries 0, 1 and 2, 3;
// int8: 0, 2 and 1, 3, as the bytes' places make them.
template <int CODES>
__device__ __forceinline__ void key_halves(uint32_t w, uint32_t& first, uint32_t& second) {
    if (CODES == FRB_E4M3) {
        halves_of_e4m3(w, first, second);
    } else {
        first = half_of_int8(w);
        second = half_of_int8(w >> 8);
    }
}

template <int CODES>
__device__ __forceinline__ void query_halves(const float (&x)[4], uint32_t& first, uint32_t& second) {
    constexpr int NEXT = CODES == FRB_E4M3 ? 1 : 2;
    first = pack_f16(x[0], x[NEXT]);
    second = pack_f16(x[3 - NEXT], x[3]);
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

// What a warp has in shared memory: a page's keys and values with their scales, and the mbarriers that announce them.
template <int HD, int VD>
struct WarpTiles {
    static constexpr int K_TILE = FRB_PAGE * HD, V_TILE = FRB_PAGE * VD, SCALES = 4 * FRB_PAGE;
    static constexpr int BYTES = D8_WARPS * (K_TILE + V_TILE + 2 * SCALES);
    uint8_t* keys;
    uint8_t* values;
    float* key_scales;
    float* value_scales;
    uint64_t* keys_full;
    uint64_t* values_full;
    uint32_t keys_parity, values_parity;
    bool keys_out, values_out;          // a copy is in flight

    __device__ __forceinline__ WarpTiles(uint8_t* base, uint64_t* bars, int warp) {
        keys = base + (size_t)warp * (K_TILE + V_TILE);
        values = keys + K_TILE;
        key_scales = reinterpret_cast<float*>(base + (size_t)D8_WARPS * (K_TILE + V_TILE) + (size_t)warp * 2 * SCALES);
        value_scales = key_scales + FRB_PAGE;
        keys_full = bars + 2 * warp;
        values_full = bars + 2 * warp + 1;
        keys_parity = values_parity = 0;
        keys_out = values_out = false;
    }
    // page kvh-th (or vh-th) head of the store's page `page`; called by all lanes
    __device__ __forceinline__ void ask_keys(const Decode8Params& p, const CUtensorMap* map, int page, int kvh, int lane) {
        if (lane == 0) {
            bar_expect(keys_full, K_TILE + SCALES);
            load_2d(keys, map, 0, (page * p.num_kv_heads + kvh) * FRB_PAGE, keys_full);
            load_row_of_scales(key_scales, p.k_scales + ((size_t)page * p.num_kv_heads + kvh) * FRB_PAGE, keys_full);
        }
        keys_out = true;
    }
    __device__ __forceinline__ void ask_values(const Decode8Params& p, const CUtensorMap* map, int page, int vh, int lane) {
        if (lane == 0) {
            bar_expect(values_full, V_TILE + SCALES);
            load_2d(values, map, 0, (page * p.v_heads + vh) * FRB_PAGE, values_full);
            load_row_of_scales(value_scales, p.v_scales + ((size_t)page * p.v_heads + vh) * FRB_PAGE, values_full);
        }
        values_out = true;
    }
    __device__ __forceinline__ bool wait_keys(int* failed) {
        if (!__all_sync(0xffffffffu, bar_wait(keys_full, keys_parity, failed))) return false;
        keys_parity ^= 1;
        keys_out = false;
        return true;
    }
    __device__ __forceinline__ bool wait_values(int* failed) {
        if (!__all_sync(0xffffffffu, bar_wait(values_full, values_parity, failed))) return false;
        values_parity ^= 1;
        values_out = false;
        return true;
    }
    // a warp that gave up leaves only when the copies that it asked for have landed (or a second limit has passed)
    __device__ __forceinline__ void leave() {
        int again = 0;
        if (keys_out) bar_wait(keys_full, keys_parity, &again);
        if (values_out) bar_wait(values_full, values_parity, &again);
    }
};

// Up to 8 NT query heads of one key head and what they have added up.  Lane 4 g + t holds, of head 2 t + c (c = 0, 1) of each tile of
// eight, the dimensions VB g .. VB g + VB - 1 of the output.
template <int HD, int VD, int NT, int CODES>
struct HeadTile {
    static constexpr int KU = HD % 64 == 0 ? 16 : 8, K_STEPS = HD / (4 * KU), K_WORDS = KU / 4;     // a lane's bytes of a key at a time
    static constexpr int VB = VD / 8, MT = VD / 16;                                                // a lane's bytes of a value; output tiles
    uint32_t q[NT][2][K_STEPS * K_WORDS];       // two registers for every word of a key (query_halves)
    float s_scale[NT][2], slope2[NT][2];        // scores to units of log2, or for a cap to units of the cap
    float gain[NT][2];                          // what scores() gives, to units of log2
    float row_max[NT][2], limit[NT][2], row_sum[NT][2];       // units of log2; a score beyond `limit` raises the maximum; row_sum: of the lane's own keys
    float inverse[NT][2];                       // 1 / U; 0 while there is no weight
    float o[NT][MT][4];

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int c = 0; c < 2; ++c) { row_max[j][c] = limit[j][c] = -INFINITY; row_sum[j][c] = 0.f; inverse[j][c] = 0.f; }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][i][e] = 0.f;
        }
    }

    // scores are what the products give times the scales, no more (and the scale keeps their order)
    static __device__ __forceinline__ bool plain(const Decode8Params& p) { return p.softcap == 0.f && !p.slopes && p.scale > 0.f; }

    // heads first_head .. first_head + heads - 1 of row b
    __device__ __forceinline__ void load_queries(const Decode8Params& p, int b, int first_head, int heads, int g, int t) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const bf16* row = p.q + ((size_t)b * p.num_heads + first_head + 8 * j + g) * HD;
            float x[K_STEPS * K_WORDS][4];
            float top = 0.f;
            bool bad = false;
#pragma unroll
            for (int s = 0; s < K_STEPS; ++s)
#pragma unroll
                for (int w = 0; w < K_WORDS; ++w) {
                    const float4 v = 8 * j + g < heads ? load4<bf16>(row + (4 * s + t) * KU + 4 * w) : make_float4(0.f, 0.f, 0.f, 0.f);
                    float (&to)[4] = x[s * K_WORDS + w];
                    to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) { top = fmaxf(top, fabsf(to[e])); bad |= !(fabsf(to[e]) < INFINITY); }
                }
            bad = ((__ballot_sync(0xffffffffu, bad) >> (4 * g)) & 15u) != 0;            // the head has an entry that is not finite: so are its scores
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = min(max(exponent_of(top), -100), 127);           // |q| 2^(14 - e) < 2^15
            const float factor = power_of_two(14 - e);
            float back = power_of_two(e - 14);
#pragma unroll
            for (int i = 0; i < K_STEPS * K_WORDS; ++i) {
#pragma unroll
                for (int d = 0; d < 4; ++d) x[i][d] *= factor;
                query_halves<CODES>(x[i], q[j][0][i], q[j][1][i]);
            }
            back *= p.softcap > 0.f ? p.scale / p.softcap : p.scale * 1.4426950408889634f;
            if (bad) back = __uint_as_float(0x7fc00000u);
            s_scale[j][0] = __shfl_sync(0xffffffffu, back, 8 * t);
            s_scale[j][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
            for (int c = 0; c < 2; ++c) gain[j][c] = plain(p) ? s_scale[j][c] : 1.f;
#pragma unroll
            for (int c = 0; c < 2; ++c)
                slope2[j][c] = p.slopes && 8 * j + 2 * t + c < heads ? p.slopes[first_head + 8 * j + 2 * t + c] * 1.4426950408889634f : 0.f;
        }
    }

    // The products of the queries with the keys of 16-key tiles i0 and i0 + 1 of a page (two at a time: the one's sums do not wait for the
    // other's), in units of s_scale: s[j][i][e] belongs to key 16 i + key_of_row(g) (+ 8 for e > 1) and head 2 t + (e & 1) of tile j.
    __device__ __forceinline__ void products(float (&s)[NT][4][4], const uint8_t* tile, int i0, int g, int t) {
        Words<KU> a[2][K_STEPS], c[2][K_STEPS];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int step = 0; step < K_STEPS; ++step) {
                const int k0 = 16 * (i0 + i) + key_of_row<VD>(g);
                a[i][step] = row_words<HD, KU>(tile, k0, (4 * step + t) * KU);
                c[i][step] = row_words<HD, KU>(tile, k0 + 8, (4 * step + t) * KU);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][i0 + i][e] = 0.f;
#pragma unroll
        for (int n = 0; n < K_STEPS * K_WORDS; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t a0, a1, a2, a3;
                key_halves<CODES>(a[i][n / K_WORDS].w[n % K_WORDS], a0, a2);
                key_halves<CODES>(c[i][n / K_WORDS].w[n % K_WORDS], a1, a3);
#pragma unroll
                for (int j = 0; j < NT; ++j) mma_f16(s[j][i0 + i], a0, a1, a2, a3, q[j][0][n], q[j][1][n]);
            }
    }

    // The scores of a page whose first key is key_base; times `gain` they are in units of log2.
    __device__ __forceinline__ void scores(const Decode8Params& p, float (&s)[NT][4][4], const uint8_t* tile, const float* scales, int key_base, int hi_key,
                                           int g, int t) {
        products(s, tile, 0, g, t);
        products(s, tile, 2, g, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k0 = 16 * i + key_of_row<VD>(g);
            const float ks0 = scales[k0], ks1 = scales[k0 + 8];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][i][e] *= e < 2 ? ks0 : ks1;
        }
        if (!plain(p)) {
            const float cap2 = p.softcap * 1.4426950408889634f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float scaled = s[j][i][e] * s_scale[j][e & 1];
                        // (the cap's minimum would turn NaN into a number)
                        const float score = cap2 > 0.f && scaled == scaled ? capped_score2(scaled, 1.f, cap2) : scaled;
                        s[j][i][e] = fmaf(slope2[j][e & 1], (float)(key_base + 16 * i + key_of_row<VD>(g) + (e < 2 ? 0 : 8) - hi_key), score);
                    }
        }
    }

    // Keys that the token may not see get no weight.
    __device__ __forceinline__ void hide(const Decode8Params& p, float (&s)[NT][4][4], int key_base, int lo_key, int hi_key, int g) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; e += 2)
                if (!key_visible(key_base + 16 * i + key_of_row<VD>(g) + 4 * e, lo_key, hi_key, p.keep_first)) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) s[j][i][e] = s[j][i][e + 1] = -INFINITY;
                }
    }

    // The running maximum follows the page's.  That is rare, so that the lanes first only ask one another whether any has a reason.
    __device__ __forceinline__ void raise(const float (&s)[NT][4][4]) {
        float top[NT][2];
        bool reason = false;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                top[j][c] = s[j][0][c];
#pragma unroll
                for (int i = 0; i < 4; ++i) top[j][c] = fmaxf(top[j][c], fmaxf(s[j][i][c], s[j][i][c + 2]));
                top[j][c] *= gain[j][c];
                reason |= top[j][c] > limit[j][c];                        // also on the first page
            }
        if (!__any_sync(0xffffffffu, reason)) return;
        float corr[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top[j][c] = fmaxf(top[j][c], __shfl_xor_sync(0xffffffffu, top[j][c], d));
                corr[j][c] = 1.f;
                if (top[j][c] > limit[j][c]) {
                    corr[j][c] = exp2_of(row_max[j][c] - top[j][c]);
                    row_max[j][c] = top[j][c];
                    limit[j][c] = top[j][c] + D8_RAISE;
                    row_sum[j][c] *= corr[j][c];
                }
            }
        rescale(corr);
    }

    __device__ __forceinline__ void rescale(const float (&corr)[NT][2]) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                o[j][i][0] *= corr[j][0]; o[j][i][1] *= corr[j][1];
                o[j][i][2] *= corr[j][0]; o[j][i][3] *= corr[j][1];
            }
    }

    // Adds the page's values, weighted.
    __device__ __forceinline__ void add_values(float (&s)[NT][4][4], const uint8_t* tile, const float* scales, int g, int t) {
        float top[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) top[j][0] = top[j][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k0 = 16 * i + key_of_row<VD>(g);
            const float vs0 = scales[k0], vs1 = scales[k0 + 8];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float weight = exp2_of(fmaf(s[j][i][e], gain[j][e & 1], -row_max[j][e & 1]));
                    row_sum[j][e & 1] += weight;
                    s[j][i][e] = weight * (e < 2 ? vs0 : vs1);
                    top[j][e & 1] = fmaxf(top[j][e & 1], s[j][i][e]);
                }
        }
        // the unit follows the largest weight times scale; rare, too
        bool reason = false;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) reason |= top[j][c] * inverse[j][c] > 32768.f || (inverse[j][c] == 0.f && top[j][c] > 0.f);
        if (__any_sync(0xffffffffu, reason)) {
            float corr[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top[j][c] = fmaxf(top[j][c], __shfl_xor_sync(0xffffffffu, top[j][c], d));
                    corr[j][c] = 1.f;
                    if (top[j][c] * inverse[j][c] > 32768.f || (inverse[j][c] == 0.f && top[j][c] > 0.f)) {
                        const int e = min(max(exponent_of(top[j][c]) - 7, -119), 119);
                        corr[j][c] = inverse[j][c] == 0.f ? 0.f : power_of_two(-e) / inverse[j][c];
                        inverse[j][c] = power_of_two(-e);
                    }
                }
            rescale(corr);
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
            const Words<VB> va = row_words<VD, VB>(tile, ka, VB * g), vb = row_words<VD, VB>(tile, kb, VB * g);
            const Words<VB> vc = row_words<VD, VB>(tile, ka + 8, VB * g), vd = row_words<VD, VB>(tile, kb + 8, VB * g);
#pragma unroll
            for (int m = 0; m < MT; ++m) {                  // rows g and g + 8: dimensions VB g + 2 m and + 1
                uint32_t a0, a1, a2, a3;
                value_halves<CODES>(va.w[m >> 1], vb.w[m >> 1], m & 1, a0, a1);
                value_halves<CODES>(vc.w[m >> 1], vd.w[m >> 1], m & 1, a2, a3);
#pragma unroll
                for (int j = 0; j < NT; ++j) mma_f16(o[j][m], a0, a1, a2, a3, b0[j], b1[j]);
            }
        }
    }

    // The sums over all of the warp's keys.
    __device__ __forceinline__ void end() {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) row_sum[j][c] += __shfl_xor_sync(0xffffffffu, row_sum[j][c], d);
    }

    // Head 8 j + 2 t + c's output entries VB g .. + VB - 1 to `row`, four or two at a time.
    __device__ __forceinline__ void store_entries(float* row, int j, int c, int g) const {
        const float unit = inverse[j][c] == 0.f ? 0.f : 1.f / inverse[j][c];          // a power of two
        if (MT % 2 == 0) {
#pragma unroll
            for (int m = 0; m < MT; m += 2)
                *reinterpret_cast<float4*>(row + VB * g + 2 * m) = make_float4(o[j][m][c] * unit, o[j][m][c + 2] * unit, o[j][m + 1][c] * unit, o[j][m + 1][c + 2] * unit);
        } else {
#pragma unroll
            for (int m = 0; m < MT; ++m) *reinterpret_cast<float2*>(row + VB * g + 2 * m) = make_float2(o[j][m][c] * unit, o[j][m][c + 2] * unit);
        }
    }
};

// Whatever lies in the places of keys that the token may not see (their weight is zero, but zero times NaN is not; int8 has no NaN).
template <int VD, int CODES>
__device__ __forceinline__ void clear_hidden(const Decode8Params& p, uint8_t* tile, float* scales, int key_base, int lo_key, int hi_key, int lane) {
    if (CODES == FRB_E4M3)
        for (int i = lane; i < FRB_PAGE * VD / 16; i += 32)
            if (!key_visible(key_base + i / (VD / 16), lo_key, hi_key, p.keep_first)) reinterpret_cast<uint4*>(tile)[i] = make_uint4(0, 0, 0, 0);
    for (int k = lane; k < FRB_PAGE; k += 32)
        if (!key_visible(key_base + k, lo_key, hi_key, p.keep_first)) scales[k] = 0.f;
    __syncwarp();
}

template <int HD, int VD>
__device__ __forceinline__ uint8_t* begin_block(uint8_t* dynamic, uint64_t* bars, int* failed) {
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * D8_WARPS; ++i) bar_init(&bars[i], 1);
        *failed = 0;
        bar_init_fence();
    }
    // an offset into the array, not an address made from a number: what is read from it is then known to be shared memory
    return dynamic + ((1024u - (smem_addr(dynamic) & 1023u)) & 1023u);
}

// ----------------------------------------------------------------------------- chunks: four pages of a key head a block

// grid (chunk, key head and tile of query heads, sequence).
template <int HD, int VD, int NT, int CODES>
__global__ void __launch_bounds__(D8_THREADS, D8_RESIDENT(HD, VD, NT))
attention_decode_8bit_chunks_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Decode8Params p) {
    // as attention_decode_tma: the copies of every page but the sequence's last go out before the kernel before this one has ended
    let_next_kernel_start();
    typedef WarpTiles<HD, VD> Tiles;
    constexpr int O_STRIDE = VD + 4;
    static_assert(NT * 8 * O_STRIDE * 4 <= Tiles::K_TILE + Tiles::V_TILE, "a warp's partial result fits into its pages");
    extern __shared__ uint8_t dynamic[];
    __shared__ uint64_t bars[2 * D8_WARPS];
    __shared__ float sm_m[D8_WARPS][8 * NT], sm_l[D8_WARPS][8 * NT];
    __shared__ int failed;
    const int chunk = blockIdx.x, kvh = blockIdx.y / p.head_tiles, tile = blockIdx.y - kvh * p.head_tiles, b = blockIdx.z;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const Sight sight = sight_of(p, b);
    if (chunk * D8_CHUNK_PAGES >= sight.count) {
        wait_for_previous_kernel();               // (were all blocks to leave without, the kernel after this one would not wait for it either)
        return;
    }
    uint8_t* base = begin_block<HD, VD>(dynamic, bars, &failed);
    Tiles tiles(base, bars, warp);
    const int n = chunk * D8_CHUNK_PAGES + warp, number = sight.number(n);
    int page = n < sight.count ? p.page_table[(size_t)p.seq_slot[b] * p.max_pages + number] : -1;
    if (page >= p.num_pages) page = -1;
    const int group = p.num_heads / p.num_kv_heads, first_head = kvh * group + tile * 8 * NT, heads = min(8 * NT, group - tile * 8 * NT);
    __syncthreads();
    const bool ahead = page >= 0 && p.early && number != sight.hi_key / FRB_PAGE;       // the kernel before this one writes to the last page
    const int vh = kvh / (p.num_kv_heads / p.v_heads);
    if (ahead) { tiles.ask_keys(p, &map_k, page, kvh, lane); tiles.ask_values(p, &map_v, page, vh, lane); }
    wait_for_previous_kernel();
    if (page >= 0 && !ahead) { tiles.ask_keys(p, &map_k, page, kvh, lane); tiles.ask_values(p, &map_v, page, vh, lane); }

    HeadTile<HD, VD, NT, CODES> rows;
    rows.begin();
    bool ok = true;
    if (page >= 0) {
        const int key_base = number * FRB_PAGE;
        const bool edge = key_base < sight.lo_key || key_base + FRB_PAGE - 1 > sight.hi_key;
        rows.load_queries(p, b, first_head, heads, g, t);
        float s[NT][4][4];
        ok = tiles.wait_keys(&failed);
        if (ok) {
            rows.scores(p, s, tiles.keys, tiles.key_scales, key_base, sight.hi_key, g, t);
            if (edge) rows.hide(p, s, key_base, sight.lo_key, sight.hi_key, g);
            rows.raise(s);
            ok = tiles.wait_values(&failed);
        }
        if (ok) {
            if (edge) clear_hidden<VD, CODES>(p, tiles.values, tiles.value_scales, key_base, sight.lo_key, sight.hi_key, lane);
            rows.add_values(s, tiles.values, tiles.value_scales, g, t);
        }
        rows.end();
    }
    if (!ok) { tiles.leave(); failed = 1; }
    __syncthreads();
    if (failed) {
        if (threadIdx.x == 0) *p.status = D8_STATUS_WAIT;
        return;
    }
    float* mine = reinterpret_cast<float*>(tiles.keys);          // [8 NT heads][O_STRIDE]
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            rows.store_entries(mine + (8 * j + 2 * t + c) * O_STRIDE, j, c, g);
            if (g == 0) { sm_m[warp][8 * j + 2 * t + c] = rows.row_max[j][c]; sm_l[warp][8 * j + 2 * t + c] = rows.row_sum[j][c]; }
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
                acc += reinterpret_cast<const float*>(base + (size_t)w * (Tiles::K_TILE + Tiles::V_TILE))[r * O_STRIDE + d] * f;
            }
        }
        const size_t row = ((size_t)b * p.num_heads + first_head + r) * p.max_chunks + chunk;
        p.part_o[row * VD + d] = acc;
        if (d == 0) { p.part_ml[row * 2] = top; p.part_ml[row * 2 + 1] = sum; }
    }
}

// ----------------------------------------------------------------------------- pieces: a warp a piece of the line of pages

// Whether row b is the row before it once more (the same token of the same sequence, as a recorded step repeats its last one).
__device__ __forceinline__ bool repeats(const Decode8Params& p, int b) {
    return b > 0 && p.seq_slot[b] == p.seq_slot[b - 1] && p.seq_pos[b] == p.seq_pos[b - 1];
}

__device__ __forceinline__ int times_repeated(const Decode8Params& p, int b) {       // of a row that repeats none: itself and its repetitions
    int n = 1;
    while (b + n < p.num_seqs && repeats(p, b + n)) ++n;
    return n;
}

// A row's places in the line, for one key head: D8_LEAD in front, since a run costs time beside its pages, and its pages, all of them as many
// times as the row is repeated, so that a piece's pages are done for all of those rows alike and repeated rows come out the same to the
// last bit.  Zero for a row that repeats another or has no pages.
__device__ __forceinline__ int places_of(const Decode8Params& p, int b) {
    if (b >= p.num_seqs || repeats(p, b)) return 0;
    const int count = sight_of(p, b).count;
    return count > 0 ? (count + D8_LEAD) * times_repeated(p, b) : 0;
}

// The same of 32 rows, b0 on, a lane each; both loads of every row at once.
__device__ __forceinline__ int places_of_rows(const Decode8Params& p, int b0, int lane) {
    const int b = b0 + lane;
    const bool there = b < p.num_seqs;
    const int slot = there ? p.seq_slot[b] : -1, position = there ? p.seq_pos[b] : -1;
    const int other = row_beside(b0, lane, p.num_seqs);
    const bool beside = other >= 0;
    const int other_slot = beside ? p.seq_slot[other] : -1, other_position = beside ? p.seq_pos[other] : -1;
    const int left_slot = __shfl_up_sync(0xffffffffu, slot, 1), left_position = __shfl_up_sync(0xffffffffu, position, 1);
    const bool repeat = there && (lane > 0 ? slot == left_slot && position == left_position : beside && slot == other_slot && position == other_position);
    const unsigned repeats_left = __ballot_sync(0xffffffffu, repeat);
    const int next_slot = __shfl_sync(0xffffffffu, other_slot, 31), next_position = __shfl_sync(0xffffffffu, other_position, 31);
    const int count = there && !repeat ? sight_from(p, slot, position).count : 0;
    if (count == 0) return 0;
    const unsigned behind = lane < 31 ? repeats_left >> (lane + 1) : 0u;
    int times = __ffs(~behind);
    if (lane + times == 32 && b0 + 32 < p.num_seqs && slot == next_slot && position == next_position) times = times_repeated(p, b);
    return (count + D8_LEAD) * times;
}

// A run: the pages [begin, end) in sight of one key head's, for one row (none where a piece lies within the repetitions of a page).  Its
// partial result is number `room` of the (row, head)'s; the first run's warp also leaves the number of all of them, in the last place's sum.
struct Run {
    Sight sight;
    int row, slot, kvh, first_head, heads, begin, end, room;
    int runs;                  // not zero: the number to leave
};

// The runs of a piece, one after the other; all lanes of a warp alike.
struct RunOrder {
    int at, piece_end, length;         // places in the line; of a piece
    int seq, times, copy;              // the row, how often it is there, which one is next
    int before, places;                // places before the row, and of one of its key heads

    // (Cut between key heads only, a piece has those that begin in it.)
    __device__ __forceinline__ bool next(const Decode8Params& p, Run& run, int per_tile) {
        for (;;) {
            if (at >= piece_end) return false;
            const int pair = (at - before) / places, pair_at = before + pair * places, pages_at = pair_at + D8_LEAD * times;
            const int run_end = p.whole ? pair_at + places : min(piece_end, pair_at + places);
            if (copy < times && run_end > pages_at && !(p.whole && at != pair_at)) {
                const int group = p.num_heads / p.num_kv_heads, tile = pair % p.head_tiles;
                run.sight = sight_of(p, seq);
                run.row = seq + copy;
                run.slot = p.seq_slot[seq];
                run.kvh = pair / p.head_tiles;
                run.first_head = run.kvh * group + tile * per_tile;
                run.heads = min(per_tile, group - tile * per_tile);
                run.begin = (max(at - pages_at, 0) + times - 1) / times;
                run.end = (run_end - pages_at + times - 1) / times;
                run.room = at / length - pages_at / length;                   // (the piece's number, and that of the first with pages)
                run.runs = run.room == 0 ? (pair_at + places - 1) / length - pages_at / length + 1 : 0;
                if (p.whole) run.room = run.runs = 0;
                ++copy;
                return true;
            }
            // on to the next key head, or the next row that has pages
            copy = 0;
            at = run_end;
            if (at < piece_end && at == before + p.num_kv_heads * p.head_tiles * places) {
                before = at;
                seq += times;
                while (seq < p.num_seqs && (places = places_of(p, seq)) == 0) ++seq;
                if (seq >= p.num_seqs) at = piece_end;                        // (not with tables that stay as they are)
                else times = times_repeated(p, seq);
            }
        }
    }
};

#define D8_ROW_GROUPS 64       // (two for a lane)
#define D8_MIN_ROOM 4          // partial results that a line cut anywhere needs room for, per (sequence, head)

template <int HD, int VD, int NT, int CODES>
__global__ void __launch_bounds__(D8_THREADS, D8_RESIDENT(HD, VD, NT))
attention_decode_8bit_pieces_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Decode8Params p) {
    let_next_kernel_start();
    typedef WarpTiles<HD, VD> Tiles;
    extern __shared__ uint8_t dynamic[];
    __shared__ uint64_t bars[2 * D8_WARPS];
    __shared__ int sums[D8_ROW_GROUPS], tops[D8_WARPS];
    __shared__ Run runs[D8_WARPS][2];
    __shared__ int failed;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int heads_in_line = p.num_kv_heads * p.head_tiles;
    uint8_t* base = begin_block<HD, VD>(dynamic, bars, &failed);

    // The line's length, from those of its rows in up to D8_ROW_GROUPS groups.
    const RowGroups in_groups = row_groups(p.num_seqs, D8_ROW_GROUPS);
    const int group_steps = in_groups.steps, groups = in_groups.count;
    int longest = 0;
    for (int i = warp; i < groups; i += D8_WARPS) {
        int sum = 0;
        for (int s = 0; s < group_steps; ++s) {
            const int places = places_of_rows(p, 32 * (i * group_steps + s), lane);
            sum += places;
            longest = max(longest, places);                 // (more than its pages: the lead in front counts, too)
        }
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0) sums[i] = sum;
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) tops[warp] = longest;
    __syncthreads();
    longest = 0;
#pragma unroll
    for (int w = 0; w < D8_WARPS; ++w) longest = max(longest, tops[w]);
    // a lane has two groups
    const int even = 2 * lane < groups ? heads_in_line * sums[2 * lane] : 0, both = even + (2 * lane + 1 < groups ? heads_in_line * sums[2 * lane + 1] : 0);
    const auto upto_lane = [&](int own) {                   // the lanes' sum up to and with this one
        int to = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int left = __shfl_up_sync(0xffffffffu, to, o);
            if (lane >= o) to += left;
        }
        return to;
    };
    const int to_both = upto_lane(both), total = __shfl_sync(0xffffffffu, to_both, 31);
    // A piece is a warp's share, at least as many places that a key head's pages lie in no more pieces than there is room for partial results
    // (less one, where their number is left).
    RunOrder order;
    order.length = max(1, (total + p.pieces - 1) / p.pieces);
    if (!p.whole) order.length = max(order.length, (longest + p.max_chunks - 3) / (p.max_chunks - 2));
    // neighbouring pieces go to different SMs: warps without a piece are then spread over all of them
    order.at = (int)min((long long)total, (long long)(warp * (int)gridDim.x + (int)blockIdx.x) * order.length);
    order.piece_end = min(total - order.at, order.length) + order.at;
    // the row that the piece begins in
    order.seq = order.before = order.places = 0;
    if (order.at < total) {
        const int pair = __ffs(__ballot_sync(0xffffffffu, order.at < to_both)) - 1;
        int upto = __shfl_sync(0xffffffffu, to_both - both, pair);
        const int first = __shfl_sync(0xffffffffu, even, pair), second = order.at >= upto + first;
        if (second) upto += first;
        const int b_end = min(p.num_seqs, (2 * pair + second + 1) * 32 * group_steps);
        for (int b0 = (2 * pair + second) * 32 * group_steps; b0 < b_end; b0 += 32) {
            const int own = heads_in_line * places_of_rows(p, b0, lane), to = upto_lane(own);
            const unsigned here = __ballot_sync(0xffffffffu, order.at < upto + to);
            if (here) {
                const int found = __ffs(here) - 1;
                order.seq = b0 + found;
                order.before = upto + __shfl_sync(0xffffffffu, to - own, found);
                order.places = __shfl_sync(0xffffffffu, own, found) / heads_in_line;
                break;
            }
            upto += __shfl_sync(0xffffffffu, to, 31);
        }
    }
    if (order.places == 0) order.at = order.piece_end;
    order.copy = 0;
    order.times = order.at < order.piece_end ? times_repeated(p, order.seq) : 0;

    Tiles tiles(base, bars, warp);
    const int v_share = p.num_kv_heads / p.v_heads;
    // the store's page of a run's page n; -1 for one that the table, or the run, does not have
    const auto page_of = [&](const Run& run, int n) {
        if (n >= run.end) return -1;
        const int page = p.page_table[(size_t)run.slot * p.max_pages + run.sight.number(n)];
        return page < p.num_pages ? page : -1;
    };
    const auto next_run = [&](int to) {                     // the next run as runs[warp][to]
        Run found;
        const bool more = order.next(p, found, 8 * NT);
        __syncwarp();
        if (lane == 0) runs[warp][to] = found;
        __syncwarp();
        return more;
    };
    int now = 0;
    bool more = next_run(now);
    int n = 0, page = -1;
    if (more) {
        const Run& run = runs[warp][now];
        n = run.begin;
        page = page_of(run, n);
        if (page >= 0 && p.early && run.sight.number(n) != run.sight.hi_key / FRB_PAGE) {      // the kernel before this one writes to the last page
            tiles.ask_keys(p, &map_k, page, run.kvh, lane);
            tiles.ask_values(p, &map_v, page, run.kvh / v_share, lane);
        }
    }
    wait_for_previous_kernel();
    if (page >= 0 && !tiles.keys_out) {
        tiles.ask_keys(p, &map_k, page, runs[warp][now].kvh, lane);
        tiles.ask_values(p, &map_v, page, runs[warp][now].kvh / v_share, lane);
    }

    HeadTile<HD, VD, NT, CODES> rows;
    bool ok = true, fresh = true;
    while (more) {
        const Run& run = runs[warp][now];
        const int key_base = run.sight.number(n) * FRB_PAGE, lo_key = run.sight.lo_key, hi_key = run.sight.hi_key;
        const bool edge = key_base < lo_key || key_base + FRB_PAGE - 1 > hi_key, last = n + 1 >= run.end, there = page >= 0;
        if (fresh) {
            rows.load_queries(p, run.row, run.first_head, run.heads, g, t);
            rows.begin();
        }
        // the page after this one: its number is there when its copy is asked for
        const int next = last ? now ^ 1 : now;
        if (last) more = next_run(next);
        n = last ? runs[warp][next].begin : n + 1;
        page = more ? page_of(runs[warp][next], n) : -1;
        float s[NT][4][4];
        if (there) {
            ok = tiles.wait_keys(&failed);
            if (!ok) break;
            rows.scores(p, s, tiles.keys, tiles.key_scales, key_base, hi_key, g, t);
        }
        __syncwarp();
        if (page >= 0) tiles.ask_keys(p, &map_k, page, runs[warp][next].kvh, lane);        // this page's keys are no longer needed
        if (there) {
            // only the pages at the window's edge, behind the first tokens and of the token itself hold keys it may not see
            if (edge) rows.hide(p, s, key_base, lo_key, hi_key, g);
            rows.raise(s);
            ok = tiles.wait_values(&failed);
            if (!ok) break;
            if (edge) clear_hidden<VD, CODES>(p, tiles.values, tiles.value_scales, key_base, lo_key, hi_key, lane);
            rows.add_values(s, tiles.values, tiles.value_scales, g, t);
            // ordinary stores into the tile come before a copy that writes there again
            if (edge) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (page >= 0) tiles.ask_values(p, &map_v, page, runs[warp][next].kvh / v_share, lane);
        if (last) {
            rows.end();
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int head = 8 * j + 2 * t + c;
                    if (head >= run.heads) continue;
                    const size_t row = ((size_t)run.row * p.num_heads + run.first_head + head) * p.max_chunks + run.room;
                    rows.store_entries(p.part_o + row * VD, j, c, g);
                    if (g == 0) {
                        *reinterpret_cast<float2*>(p.part_ml + row * 2) = make_float2(rows.row_max[j][c], rows.row_sum[j][c]);
                        if (run.runs > 0) p.part_ml[(row + p.max_chunks - 1) * 2 + 1] = (float)run.runs;           // (the first run: room 0)
                    }
                }
        }
        fresh = last;
        now = next;
    }
    if (!ok) {
        tiles.leave();
        failed = 1;
        if (lane == 0) *p.status = D8_STATUS_WAIT;
    }
}

// ----------------------------------------------------------------------------- the join

// Maximum (units of log2), sum and unnormalised output entries of some partial results; a lane has N entries side by side.
template <int N>
struct Joined {
    float top = -INFINITY, sum = 0.f, acc[N] = {};
    __device__ __forceinline__ void add(float other_top, float other_sum, const float (&other)[N]) {
        if (other_sum == 0.f) return;                 // no key (a sum that is not a number is none of these)
        const float both = fmaxf(top, other_top), fa = sum == 0.f ? 0.f : exp2f(top - both), fb = exp2f(other_top - both);
        top = both;
        sum = sum * fa + other_sum * fb;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = acc[e] * fa + other[e] * fb;
    }
};

template <int N>
__device__ __forceinline__ void load_entries(const float* from, float (&to)[N]) {
    if constexpr (N == 4) {
        const float4 v = *reinterpret_cast<const float4*>(from);
        to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
    } else if constexpr (N == 2) {
        const float2 v = *reinterpret_cast<const float2*>(from);
        to[0] = v.x; to[1] = v.y;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) to[e] = from[e];
    }
}

// The partial results share, share + shares, ... of a (row, head) in that order: a lane weighs one of 32, then the warp adds their entries.
// The first entries are asked for before the number of partial results is known: places without one are read and not used.
template <int N>
__device__ __forceinline__ Joined<N> joined_parts(const Decode8Params& p, size_t row0, int pages, int lane, int share, int shares) {
    constexpr int AT_ONCE = 4, VD = 32 * N;
    Joined<N> all;
    const float* entries = p.part_o + row0 * VD + N * lane;
    float first[AT_ONCE][N];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
        if (share + u * shares < p.max_chunks) load_entries<N>(entries + (size_t)(share + u * shares) * VD, first[u]);
    int count = p.max_chunks;
    for (int c0 = share; c0 < count; c0 += 32 * shares) {
        const int mine = c0 + lane * shares;
        const float2 ml = mine < p.max_chunks ? *reinterpret_cast<const float2*>(p.part_ml + (row0 + mine) * 2) : make_float2(0.f, 0.f);
        if (c0 == share) count = p.whole ? min(pages, 1) : p.pieces == 0 ? (pages + D8_CHUNK_PAGES - 1) / D8_CHUNK_PAGES
                               : pages > 0 ? min((int)p.part_ml[(row0 + p.max_chunks - 1) * 2 + 1], p.max_chunks) : 0;
        const bool has = mine < count && ml.y != 0.f;
        const unsigned some = __ballot_sync(0xffffffffu, has);
        if (some == 0) continue;
        const float top = fmaxf(all.top, warp_max(has ? ml.x : -INFINITY)), keep = all.sum == 0.f ? 0.f : exp2f(all.top - top);
        const float weight = has ? exp2f(ml.x - top) : 0.f;
        all.top = top;
        all.sum = all.sum * keep + warp_sum(has ? ml.y * weight : 0.f);
#pragma unroll
        for (int e = 0; e < N; ++e) all.acc[e] *= keep;
        const int here = 32 - __clz(some);
#pragma unroll 1
        for (int u0 = 0; u0 < here; u0 += AT_ONCE) {
            float part[AT_ONCE][N];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                if (c0 == share && u0 == 0) {
#pragma unroll
                    for (int e = 0; e < N; ++e) part[u][e] = first[u][e];
                } else if (u0 + u < here) load_entries<N>(entries + (size_t)(c0 + (u0 + u) * shares) * VD, part[u]);
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const float f = __shfl_sync(0xffffffffu, weight, u0 + u);
                if (some >> (u0 + u) & 1)
#pragma unroll
                    for (int e = 0; e < N; ++e) all.acc[e] += part[u][e] * f;
            }
        }
    }
    return all;
}

#define D8_JOIN_WARPS 8

// grid (8 / shares output heads, sequence): `shares` warps a (sequence, head), a lane VD / 32 entries side by side.  What bounds it is latency, or for many
// sequences the partial results' bytes.  A (sequence, head) without any key gives zeros, with a sink or not.
template <int VD>
__global__ void __launch_bounds__(32 * D8_JOIN_WARPS, 3) attention_decode_8bit_join_kernel(Decode8Params p, int shares_log2) {
    constexpr int N = VD / 32;
    __shared__ Joined<N> others[D8_JOIN_WARPS][32];
    const int heads = p.lam ? p.num_heads / 2 : p.num_heads, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int shares = 1 << shares_log2, share = warp & (shares - 1), head = (int)(blockIdx.x * D8_JOIN_WARPS + warp) >> shares_log2;
    const Sight sight = sight_of(p, b);                        // from the step's tables, which were there before the kernel before this one began
    wait_for_previous_kernel();
    // (The kernel after this one starts no earlier: were it attention once more, its blocks would take the SMs' room unevenly while pieces are
    // still being done; 32 sequences of 4,096 keys took 59 us, with this 54.)
    let_next_kernel_start();
    if (sight.cut && threadIdx.x == 0) atomicExch(p.status, D8_STATUS_TOO_LONG);               // keys were left out
    const auto joined = [&](int query_head) {
        Joined<N> all;
        if (head < heads) all = joined_parts<N>(p, ((size_t)b * p.num_heads + query_head) * p.max_chunks, sight.count, lane, share, shares);
        if (shares > 1) {
            __syncthreads();                                   // (read from an earlier call)
            others[warp][lane] = all;
            __syncthreads();
            if (share == 0)
                for (int s = 1; s < shares; ++s) all.add(others[warp + s][lane].top, others[warp + s][lane].sum, others[warp + s][lane].acc);
        }
        return all;
    };
    float result[N];
    if (p.lam) {
        const int group = p.num_heads / p.num_kv_heads, pair = head / group, first = 2 * pair * group + (head - pair * group);
        const Joined<N> one = joined(first), two = joined(first + group);
        float squares = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            result[e] = (one.sum == 0.f ? 0.f : one.acc[e] / one.sum) - *p.lam * (two.sum == 0.f ? 0.f : two.acc[e] / two.sum);
            squares += result[e] * result[e];
        }
        const float rms = sqrtf(warp_sum(squares) / (float)VD + p.diff_eps);
#pragma unroll
        for (int e = 0; e < N; ++e) result[e] = result[e] / rms * p.diff_factor;
    } else {
        Joined<N> all = joined(head);
        if (p.sinks && all.sum != 0.f && head < heads) {
            const float nothing[N] = {};
            all.add(p.sinks[head] * 1.4426950408889634f, 1.f, nothing);      // a term of the denominator without a value
        }
        const float inverse = all.sum == 0.f ? 0.f : 1.f / all.sum;
#pragma unroll
        for (int e = 0; e < N; ++e) result[e] = all.sum == 0.f ? 0.f : all.acc[e] * inverse;
    }
    if (share != 0 || head >= heads) return;
    bf16* out = p.out + ((size_t)b * heads + head) * VD + N * lane;
    if constexpr (N % 2 == 0) {
        uint32_t two[N / 2];
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(result[e], result[e + 1]);
            two[e / 2] = *reinterpret_cast<const uint32_t*>(&v);
        }
        if constexpr (N == 4) *reinterpret_cast<uint2*>(out) = make_uint2(two[0], two[1]);
        else *reinterpret_cast<uint32_t*>(out) = two[0];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) out[e] = __float2bfloat16_rn(result[e]);
    }
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
static void launch_decode_8bit(const CUtensorMap& map_k, const CUtensorMap& map_v, const Decode8Params& p, cudaStream_t stream) {
    const size_t smem = (size_t)WarpTiles<HD, VD>::BYTES + 1024;
    const bool pieces = p.pieces > 0;
    auto kernel = pieces ? attention_decode_8bit_pieces_kernel<HD, VD, NT, CODES> : attention_decode_8bit_chunks_kernel<HD, VD, NT, CODES>;
    const dim3 grid = pieces ? dim3((p.pieces + D8_WARPS - 1) / D8_WARPS) : dim3(p.max_chunks, p.num_kv_heads * p.head_tiles, p.num_seqs);
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    launch_dependent_resident(p.early ? D8_RESIDENT(HD, VD, NT) : 1, kernel, grid, dim3(D8_THREADS), smem, stream, map_k, map_v, p);
}

// max_chunks: chunks of 256 keys of the longest sequence (or more); part_o and part_ml hold as many partial results per (sequence, head).
// num_pages: pages of the store.  max_pieces: 0, or into how many pieces (warps) the work is cut, whatever its size.  pages_final: every page but a
// sequence's newest was written by kernels that had ended when the kernel before this one began.  status: one int on the device.
FRB_API int frb_attention_decode_8bit(const void* q, const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales,
                                      int codes, int num_pages, const int* page_table, int num_slots, int max_pages, const int* seq_pos,
                                      const int* seq_slot, float* part_o, float* part_ml, void* out, int num_seqs, int num_heads,
                                      int num_kv_heads, int v_heads, int head_dim, int v_dim, float scale, int window, int chunk,
                                      int keep_first, int max_chunks, int max_pieces, const float* slopes, const float* sinks,
                                      float softcap, const float* lam, float diff_eps, float diff_factor, int pages_final,
                                      int* status, cudaStream_t stream) {
    if (num_seqs == 0) return 0;
    FRB_CHECK_ARG(num_seqs > 0 && num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0 && v_heads > 0 && num_kv_heads % v_heads == 0,
                  "attention_decode_8bit: %d sequences, %d heads over %d key heads and %d value heads", num_seqs, num_heads, num_kv_heads, v_heads);
    FRB_CHECK_ARG(codes == FRB_E4M3 || codes == FRB_INT8, "attention_decode_8bit: codes of type %d", codes);
    FRB_CHECK_ARG(num_pages > 0 && num_slots > 0 && max_pages > 0 && max_pages < (1 << 25), "attention_decode_8bit: %d pages, %d slots of %d",
                  num_pages, num_slots, max_pages);
    FRB_CHECK_ARG((long long)num_pages * num_kv_heads * FRB_PAGE < (1ll << 31), "attention_decode_8bit: %d pages of %d heads exceed a tensor map's rows",
                  num_pages, num_kv_heads);
    FRB_CHECK_ARG(max_chunks >= 1 && max_chunks < (1 << 23) && max_pieces >= 0 && max_pieces <= (1 << 24),
                  "attention_decode_8bit: %d chunks, %d pieces", max_chunks, max_pieces);
    FRB_CHECK_ARG(window >= 0 && chunk >= 0 && keep_first >= 0 && !(keep_first > 0 && chunk > 0),
                  "attention_decode_8bit: a window of %d, chunks of %d, %d first tokens", window, chunk, keep_first);
    FRB_CHECK_ARG(!lam || (num_kv_heads == 2 * v_heads && !sinks), "attention_decode_8bit: two maps per head need two key heads a value head and no sinks");
    const auto aligned = [](const void* ptr, uintptr_t bytes) { return ((uintptr_t)ptr & (bytes - 1)) == 0; };
    FRB_CHECK_ARG(aligned(q, 8) && aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(k_scales, 16) && aligned(v_scales, 16) &&
                  aligned(part_o, 16) && aligned(part_ml, 8) && aligned(out, 8),
                  "attention_decode_8bit: queries, maxima and outputs start on 8 bytes, codes, scales and partial outputs on 16");
    const int group = num_heads / num_kv_heads, per_block = group <= 8 ? 8 : 16, head_tiles = (group + per_block - 1) / per_block;
    FRB_CHECK_ARG(num_seqs <= 65535 && (long long)num_kv_heads * head_tiles <= 65535, "attention_decode_8bit: %d sequences of %d heads exceed the grid",
                  num_seqs, num_heads);
    Decode8Params p;
    p.q = (const bf16*)q; p.k_scales = k_scales; p.v_scales = v_scales; p.page_table = page_table; p.seq_pos = seq_pos; p.seq_slot = seq_slot;
    p.part_o = part_o; p.part_ml = part_ml; p.out = (bf16*)out; p.slopes = slopes; p.sinks = sinks; p.lam = lam; p.status = status;
    p.scale = scale; p.softcap = softcap > 0.f ? softcap : 0.f; p.diff_eps = diff_eps; p.diff_factor = diff_factor; p.window = window;
    p.chunk = chunk; p.keep_first = window > 0 ? keep_first : 0; p.max_pages = max_pages; p.num_slots = num_slots; p.num_pages = num_pages;
    p.num_heads = num_heads; p.num_kv_heads = num_kv_heads; p.v_heads = v_heads; p.num_seqs = num_seqs; p.max_chunks = max_chunks;
    p.head_tiles = head_tiles;
    // Chunks where two waves of blocks hold all that there may be.  Measured on a B200 with 48 heads on 8 key heads of 128, sequences x keys, microseconds
    // with the join, chunks | pieces: 64 blocks (1 x 2048) 6.5 | 17.0; 256 (1 x 8192) 10.0 | 16.5; 512 (4 x 4096) 18.0 | 17.5, (8 x 2048) 17.8 | 19.0;
    // 1,024 (8 x 4096) 25.7 | 21.3; 2,048 (8 x 8192) 40.9 | 31.2, (128 x 512, cut between key heads) 44.9 | 37.2; 4,096 (32 x 4096) 69.9 | 53.7,
    // (1 x 131072) 78.9 | 53.6; 8,192 blocks with a page each (1024 x 40) 142 | 76.  Heads of 64: 1,024 (8 x 4096) 16.3 | 17.5, 2,048 (8 x 8192)
    // 24.3 | 21.1, (128 x 512) 27.0 | 31.9, 4,096 (32 x 4096) 40.0 | 35.2.  The rule counts the blocks that there may be (max_chunks), not the pages that are in
    // sight: it takes pieces for the 128 x 512 of heads of 64, and for a window far shorter than what max_chunks stands for.
    const int resident = D8_RESIDENT(head_dim, v_dim, per_block / 8) * frb_sm_count();
    const long long chunks = (long long)num_seqs * num_kv_heads * head_tiles * max_chunks;
    const bool countable = chunks * D8_CHUNK_PAGES < (1ll << 30);
    p.pieces = !countable ? 0 : max_pieces > 0 ? max_pieces : chunks > 2ll * resident ? resident * D8_WARPS : 0;
    p.whole = p.pieces > 0 && max_chunks < D8_MIN_ROOM;
    static const int early = [] { const char* v = getenv("FIELDRUN_B200_ATTENTION_EARLY"); return !(v && v[0] == '0'); }();
    p.early = early && pages_final;
    CUtensorMap map_k, map_v;
    FRB_CHECK_ARG(map_code_rows(&map_k, k_codes, (uint64_t)num_pages * num_kv_heads * FRB_PAGE, head_dim) &&
                  map_code_rows(&map_v, v_codes, (uint64_t)num_pages * v_heads * FRB_PAGE, v_dim),
                  "attention_decode_8bit: head_dim %d with value heads of %d: cuTensorMapEncodeTiled failed or is not available", head_dim, v_dim);
    const int out_heads = lam ? num_heads / 2 : num_heads;
    // the join: more warps a (sequence, head) while that leaves SMs idle and each has some partial results
    int shares_log2 = 0;
    while ((1 << shares_log2) < D8_JOIN_WARPS && ((long long)out_heads * num_seqs << shares_log2) <= 6 * frb_sm_count() && max_chunks >= 8 << shares_log2) ++shares_log2;
    const dim3 join_grid(((out_heads << shares_log2) + D8_JOIN_WARPS - 1) / D8_JOIN_WARPS, num_seqs), join_block(32 * D8_JOIN_WARPS);
#define FRB_LAUNCH_DECODE8(HD, VD)                                                                                                  \
    if (per_block == 8 && codes == FRB_E4M3) launch_decode_8bit<HD, VD, 1, FRB_E4M3>(map_k, map_v, p, stream);                \
    else if (per_block == 8) launch_decode_8bit<HD, VD, 1, FRB_INT8>(map_k, map_v, p, stream);                                \
    else if (codes == FRB_E4M3) launch_decode_8bit<HD, VD, 2, FRB_E4M3>(map_k, map_v, p, stream);                             \
    else launch_decode_8bit<HD, VD, 2, FRB_INT8>(map_k, map_v, p, stream);                                                    \
    launch_dependent_resident(early ? 4 : 1, attention_decode_8bit_join_kernel<VD>, join_grid, join_block, 0, stream, p, shares_log2)
    FRB_8BIT_SIZES("attention_decode_8bit", head_dim, v_dim, FRB_LAUNCH_DECODE8);
#undef FRB_LAUNCH_DECODE8
    FRB_RETURN_LAUNCH("attention_decode_8bit");
}

FRB_API int frb_attention_decode_8bit_packed(const void* packed, cudaStream_t stream) { return call_packed(frb_attention_decode_8bit, packed, stream); }
