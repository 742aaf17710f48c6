// Rows written into a cache of 8-bit pages, and pages read back.
//
// qkv_prepare_8bit does what qkv_prepare does (bias, norms of queries and keys, rotation, the queries' temperature,
// src/minimax.rs:136-150, 253-268) and stores keys and values as codes with a scale a row (cache_8bit.cuh): the counterpart of
// the reference's row quantiser for its 8-bit cache (src/minimax.rs:291-347).  cache_read_8bit gives the rows of chosen pages
// back as bfloat16 pages in the layout that the prompt attention kernels read.
#include "cache_8bit.cuh"
#include "tma.cuh"

using namespace frb_8bit;
using namespace frb_tma;

struct Write8Params {
    const void* qkv;          // [T, (nh + nkv) * hd + nvh * vd]; without the value columns where the values are the keys
    const float* bias;        // as wide as a row, added before anything else, or null
    const void* q_weight;     // [nh * hd], or with per_head [hd]; null: no norm
    const void* k_weight;
    const float* cos_table;   // [positions, rotary_dim / 2]
    const float* sin_table;
    const int* tok_pos;       // [T]
    const int* tok_slot;      // [T]
    const int* page_table;    // [slots, max_pages]
    bf16* q_out;              // [T, nh, hd]
    uint8_t* k_codes;         // [pages, nkv, 64, hd]
    float* k_scales;          // [pages, nkv, 64]
    uint8_t* v_codes;         // [pages, nvh, 64, vd]
    float* v_scales;
    float eps, q_temp_coef;
    int q_temp_every, num_heads, num_kv_heads, num_v_heads, rotary_dim, interleaved, max_pages, num_slots, num_pages, table_positions;
    int per_head, tables_final, row_width, v_from, codes, in_f32, weight_f32, num_tokens, stages, angles_by_four;
    int* status;
};

__device__ __forceinline__ float4 four_of(const void* base, size_t at, int is_f32) {
    return is_f32 ? load4<float>(reinterpret_cast<const float*>(base) + at) : load4<bf16>(reinterpret_cast<const bf16*>(base) + at);
}

// Four entries of a row in shared memory, with the bias.
template <bool LEAN>
__device__ __forceinline__ float4 entries_of(const Write8Params& p, const uint8_t* row, int column) {
    if (LEAN) return *reinterpret_cast<const float4*>(row + 4 * (size_t)column);
    const float4 a = four_of(row, column, p.in_f32);
    if (!p.bias) return a;
    const float4 b = *reinterpret_cast<const float4*>(p.bias + column);
    return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// The largest of `v` over runs of LANES lanes, and the sum.
template <int LANES>
__device__ __forceinline__ uint32_t run_max(uint32_t v) {
    if constexpr (LANES == 32) {
        return __reduce_max_sync(0xffffffffu, v);
    } else {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    }
}

template <int LANES>
__device__ __forceinline__ float run_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float4 times(float4 a, float f) { return make_float4(a.x * f, a.y * f, a.z * f, a.w * f); }
__device__ __forceinline__ float4 times(float4 a, float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); }
__device__ __forceinline__ float squares(float4 a) { return a.x * a.x + a.y * a.y + a.z * a.z + a.w * a.w; }
__device__ __forceinline__ uint32_t largest(float4 a) {
    return max(max(magnitude_bits(a.x), magnitude_bits(a.y)), max(magnitude_bits(a.z), magnitude_bits(a.w)));
}

// How a row's dimensions turn: not at all, in pairs of neighbours within a lane's four, in pairs of whole fours, or in any other pairs.
enum TurnKind { TURN_NONE, TURN_NEIGHBOURS, TURN_FOURS, TURN_ANY };

// The lane's part of a head's rotation: cosines and sines for the four dimensions from `dim` on (1 and 0 where nothing turns).
//     a' = a c - b s ; b' = b c + a s   (src/minimax.rs:78-81)
struct Turn {
    float4 cos, sin;

    __device__ __forceinline__ void load(const Write8Params& p, int kind, int position, int dim) {
        cos = make_float4(1.f, 1.f, 1.f, 1.f);
        sin = make_float4(0.f, 0.f, 0.f, 0.f);
        const int rot = p.rotary_dim, half = rot / 2;
        if (dim >= rot) return;
        const size_t row = (size_t)min(max(position, 0), p.table_positions - 1) * half;
        if (kind == TURN_FOURS) {
            const bool lower = dim < half;
            const size_t at = row + (lower ? dim : dim - half);
            cos = *reinterpret_cast<const float4*>(p.cos_table + at);
            sin = *reinterpret_cast<const float4*>(p.sin_table + at);
            if (lower) sin = make_float4(-sin.x, -sin.y, -sin.z, -sin.w);
        } else if (kind == TURN_NEIGHBOURS) {
            const size_t at = row + (dim >> 1);
            const float c0 = p.cos_table[at], c1 = p.cos_table[at + 1], s0 = p.sin_table[at], s1 = p.sin_table[at + 1];
            cos = make_float4(c0, c0, c1, c1);
            sin = make_float4(-s0, s0, -s1, s1);
        } else {
            float* c = &cos.x;
            float* s = &sin.x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = dim + e;
                if (d >= rot) continue;
                const bool lower = p.interleaved ? (d & 1) == 0 : d < half;
                const size_t at = row + (p.interleaved ? d >> 1 : lower ? d : d - half);
                c[e] = p.cos_table[at];
                s[e] = lower ? -p.sin_table[at] : p.sin_table[at];
            }
        }
    }
    __device__ __forceinline__ float4 with(float4 a, float4 b) const {                    // b: the partners
        return make_float4(a.x * cos.x + b.x * sin.x, a.y * cos.y + b.y * sin.y, a.z * cos.z + b.z * sin.z, a.w * cos.w + b.w * sin.w);
    }
    // from: TURN_FOURS, the partners' lane
    template <int KIND, int LANES>
    __device__ __forceinline__ float4 of(const Write8Params& p, float4 a, int dim, int lane, int from) const {
        if (KIND == TURN_NONE) return a;
        if (KIND == TURN_NEIGHBOURS) return with(a, make_float4(a.y, a.x, a.w, a.z));
        if (KIND == TURN_FOURS)
            return with(a, make_float4(__shfl_sync(0xffffffffu, a.x, from), __shfl_sync(0xffffffffu, a.y, from), __shfl_sync(0xffffffffu, a.z, from),
                                       __shfl_sync(0xffffffffu, a.w, from)));
        return with(a, partners(a, p.rotary_dim, p.interleaved, dim, lane & ~(LANES - 1)));
    }
    static __device__ __forceinline__ float4 partners(float4 a, int rot, int interleaved, int dim, int first_lane) {
        const int half = rot / 2;
        float r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = dim + e, partner = d >= rot ? d : interleaved ? d ^ 1 : d < half ? d + half : d - half;
            const int at = first_lane + (partner >> 2);
            const float x = __shfl_sync(0xffffffffu, a.x, at), y = __shfl_sync(0xffffffffu, a.y, at);
            const float z = __shfl_sync(0xffffffffu, a.z, at), w = __shfl_sync(0xffffffffu, a.w, at);
            r[e] = (partner & 2) == 0 ? ((partner & 1) == 0 ? x : y) : ((partner & 1) == 0 ? z : w);
        }
        return make_float4(r[0], r[1], r[2], r[3]);
    }
};

// A row's codes and scale, by the run of LANES lanes that hold it; nothing from lanes that do not `store`.
template <int LANES>
__device__ __forceinline__ void store_codes(float4 a, bool store, uint8_t* codes, float* scale, int dim, int type) {
    const uint32_t top = run_max<LANES>(largest(a));
    if (!store) return;
    float factor, s;
    row_scale(top, type, factor, s);
    *reinterpret_cast<uint32_t*>(codes) = four_codes(a, factor, type);
    if (dim == 0) *scale = s;
}

#define WRITE8_STATUS_WAIT 9           // a wait gave up

// Where a token's row lies and goes to.
struct Place8 {
    const uint8_t* row;        // in shared memory
    bf16* q;
    int page, in_page;
};

// The queries and keys of a row: a warp takes spans of 32 lanes, four entries a lane (a head of 128, two of 64, four of 32; a head of 96 leaves
// eight lanes idle).  of_q and of_k: what multiplies all entries alike (the root of a whole row's statistic, the queries' temperature).
template <int HD, int KIND, bool LEAN>
__device__ __forceinline__ void write_queries_and_keys(const Write8Params& p, const Place8& at, const Turn& turn, float of_q, float of_k, float4 head_wq,
                                                       float4 head_wk) {
    constexpr int LANES = HD == 96 ? 32 : HD / 4, SPAN = 32 / LANES * HD;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, dim = 4 * (lane % LANES);
    const int q_width = p.num_heads * HD, width = q_width + p.num_kv_heads * HD, half = p.rotary_dim / 2;
    const int from = KIND == TURN_FOURS && dim < p.rotary_dim ? lane + (dim < half ? half / 4 : -half / 4) : lane;
    const bool weights = p.q_weight != nullptr && !p.per_head, idle = HD == 96 && lane >= 24;
    const auto value = [&](int column, bool mine, bool is_q) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        if (mine) {
            a = entries_of<LEAN>(p, at.row, column);
            if (weights) a = times(a, is_q ? four_of(p.q_weight, column, LEAN || p.weight_f32) : four_of(p.k_weight, column - q_width, LEAN || p.weight_f32));
        }
        float f = is_q ? of_q : of_k;
        if (p.per_head) {
            f *= rsqrtf(run_sum<LANES>(squares(a)) * (1.f / (float)HD) + p.eps);
            a = times(a, is_q ? head_wq : head_wk);
        }
        return turn.template of<KIND, LANES>(p, times(a, f), dim, lane, from);
    };
    int first = warp * SPAN;
#pragma unroll 4
    for (; first + SPAN <= q_width; first += warps * SPAN) {      // spans of queries alone
        const float4 a = value(first + 4 * lane, !idle, true);
        if (!idle) store4<bf16>(at.q + first + 4 * lane, a);
    }
    for (; first < width; first += warps * SPAN) {                // of keys, or of both
        const int column = first + 4 * lane;
        const bool mine = !idle && column < width, is_q = column < q_width;
        const float4 a = value(column, mine, is_q);
        if (mine && is_q) store4<bf16>(at.q + column, a);
        if (at.page < 0) continue;
        const size_t to = ((size_t)at.page * p.num_kv_heads + (column - q_width) / HD) * FRB_PAGE + at.in_page;
        store_codes<LANES>(a, mine && !is_q, p.k_codes + to * HD + dim, p.k_scales + to, dim, p.codes);
    }
}

// A block takes a token at a time.  Its row comes into shared memory by one copy, the next token's while the present one is worked on.  A head's
// statistic, its largest entry and its pairs of dimensions are exchanges between lanes; only the statistics over whole rows need the
// block.  What bounds it for prompts is the rows' bytes (4 an entry in, 2 a query entry and 1 a key or value entry out) and its
// instructions, 115 a warp and 128 entries.  (Rows held in registers, eight spans a warp unrolled, took three times as many.)  Measured on a B200 with
// MiniMax-M2's rows of 8,192 entries: 1 token 4.3 us, 64 tokens 4.5 us, a prompt of 2,048 31 us (3.1 TB/s; issue slots 46 % busy, the loads of norm
// weights and angles the largest stall).
// LEAN: rows and weights in float32, no bias.  (The other form, for everything else, spills 68 to 108 bytes a thread; it was not timed.)
template <int HD, int VD, int THREADS, int RESIDENT, bool LEAN>
__global__ void __launch_bounds__(THREADS, RESIDENT) qkv_prepare_8bit_kernel(Write8Params p) {
    let_next_kernel_start();
    extern __shared__ __align__(16) uint8_t rows[];
    __shared__ uint64_t full[2];
    __shared__ float sums[2][2][32];
    __shared__ int failed;
    constexpr int K_LANES = HD == 96 ? 32 : HD / 4, V_LANES = VD == 96 ? 32 : VD / 4, V_SPAN = 32 / V_LANES * VD;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int q_width = p.num_heads * HD, qk_width = q_width + p.num_kv_heads * HD, v_width = p.num_v_heads * VD;
    const int k_dim = 4 * (lane % K_LANES), v_dim = 4 * (lane % V_LANES);
    const bool whole = !p.per_head && p.q_weight;
    const int rot = p.rotary_dim;
    const int kind = rot == 0 ? TURN_NONE : p.interleaved ? (rot % 4 == 0 ? TURN_NEIGHBOURS : TURN_ANY) : rot % 8 == 0 && p.angles_by_four ? TURN_FOURS : TURN_ANY;
    int t = blockIdx.x, pos = 0, next_pos = 0, next_slot = 0;
    Place8 at = {rows, p.q_out, -1, 0};
    Turn turn;
    const auto next_place = [&](int token) {
        if (token < p.num_tokens) { next_pos = p.tok_pos[token]; next_slot = p.tok_slot[token]; }
    };
    // the token's page and angles, and the next one's place; a position, slot or page that does not exist writes nothing
    const auto tables = [&] {
        pos = next_pos;
        const int slot = next_slot;
        at.page = -1;
        if (pos >= 0 && pos / FRB_PAGE < p.max_pages && slot >= 0 && slot < p.num_slots)
            at.page = p.page_table[(size_t)slot * p.max_pages + pos / FRB_PAGE];
        if (at.page >= p.num_pages) at.page = -1;
        at.in_page = pos & (FRB_PAGE - 1);
        turn.load(p, kind, pos, k_dim);
        next_place(t + gridDim.x);
    };
    const uint32_t row_bytes = (uint32_t)p.row_width * (LEAN || p.in_f32 ? 4 : 2);
    const auto ask = [&](int token, int stage) {
        bar_expect(&full[stage], row_bytes);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(smem_addr(rows + (size_t)stage * row_bytes)), "l"(reinterpret_cast<const uint8_t*>(p.qkv) + (size_t)token * row_bytes),
                     "r"(row_bytes), "r"(smem_addr(&full[stage])) : "memory");
    };
    if (threadIdx.x == 0) {
        bar_init(&full[0], 1);
        bar_init(&full[1], 1);
        failed = 0;
        bar_init_fence();
    }
    // positions, slots, pages and angles that were there before the kernel before this one began; the norms' weights always were
    if (p.tables_final) {
        next_place(t);
        tables();
    }
    if (whole) {
        const int line = 128 / (p.weight_f32 ? 4 : 2);
        for (int i = threadIdx.x * line; i < qk_width; i += blockDim.x * line) {
            const size_t from = (size_t)(i < q_width ? i : i - q_width) * (p.weight_f32 ? 4 : 2);
            asm volatile("prefetch.global.L1 [%0];" ::"l"(reinterpret_cast<const uint8_t*>(i < q_width ? p.q_weight : p.k_weight) + from));
        }
    }
    float4 head_wq, head_wk;                                // a norm per head has the same weights for every head
    head_wq = head_wk = make_float4(1.f, 1.f, 1.f, 1.f);
    if (p.per_head && k_dim < HD) {
        head_wq = four_of(p.q_weight, k_dim, p.weight_f32);
        head_wk = four_of(p.k_weight, k_dim, p.weight_f32);
    }
    __syncthreads();
    wait_for_previous_kernel();
    if (threadIdx.x == 0)
        for (int s = 0; s < p.stages; ++s)
            if (t + s * (int)gridDim.x < p.num_tokens) ask(t + s * gridDim.x, s);
    if (!p.tables_final) {
        next_place(t);
        tables();
    }

    for (int n = 0;; ++n) {
        const int stage = p.stages == 2 ? n & 1 : 0;
        at.row = rows + (size_t)stage * row_bytes;
        at.q = p.q_out + (size_t)t * q_width;
        const bool ok = bar_wait(&full[stage], (uint32_t)(p.stages == 2 ? n >> 1 : n) & 1u, &failed);
        // statistics of whole rows
        if (whole) {
            float ssq = 0.f, ssk = 0.f;
            int i = 4 * threadIdx.x;
#pragma unroll 4
            for (; i < q_width; i += 4 * blockDim.x) ssq += squares(entries_of<LEAN>(p, at.row, i));
            for (; i < qk_width; i += 4 * blockDim.x) ssk += squares(entries_of<LEAN>(p, at.row, i));
            ssq = warp_sum(ssq);
            ssk = warp_sum(ssk);
            if (lane == 0) { sums[n & 1][0][warp] = ssq; sums[n & 1][1][warp] = ssk; }
        }
        if (__syncthreads_or(!ok)) {                        // leave when the copies have landed (or a second limit has passed)
            if (threadIdx.x == 0) {
                *p.status = WRITE8_STATUS_WAIT;
                int again = 0;
                for (int s = 0; s < p.stages; ++s) {
                    const int uses = p.stages == 2 ? (n + (s == stage ? 0 : 1)) >> 1 : n;
                    if (t + (s == stage ? 0 : 1) * (int)gridDim.x < p.num_tokens) bar_wait(&full[s], (uint32_t)uses & 1u, &again);
                }
            }
            __syncthreads();
            return;
        }
        float of_q = 1.f, of_k = 1.f;
        if (whole) {
            float ssq = 0.f, ssk = 0.f;
            if (warps <= 8) {
                for (int w = 0; w < warps; ++w) { ssq += sums[n & 1][0][w]; ssk += sums[n & 1][1][w]; }
            } else {
                ssq = warp_sum(lane < warps ? sums[n & 1][0][lane] : 0.f);
                ssk = warp_sum(lane < warps ? sums[n & 1][1][lane] : 0.f);
            }
            of_q = rsqrtf(ssq / (float)q_width + p.eps);
            of_k = rsqrtf(ssk / (float)(qk_width - q_width) + p.eps);
        }
        if (p.q_temp_coef != 0.f) of_q *= 1.f + p.q_temp_coef * logf((float)((pos + 1) / p.q_temp_every) + 1.f);
        if (kind == TURN_FOURS) write_queries_and_keys<HD, TURN_FOURS, LEAN>(p, at, turn, of_q, of_k, head_wq, head_wk);
        else if (kind == TURN_NONE) write_queries_and_keys<HD, TURN_NONE, LEAN>(p, at, turn, of_q, of_k, head_wq, head_wk);
        else if (kind == TURN_NEIGHBOURS) write_queries_and_keys<HD, TURN_NEIGHBOURS, LEAN>(p, at, turn, of_q, of_k, head_wq, head_wk);
        else write_queries_and_keys<HD, TURN_ANY, LEAN>(p, at, turn, of_q, of_k, head_wq, head_wk);
        if (at.page >= 0)
            for (int first = warp * V_SPAN; first < v_width; first += warps * V_SPAN) {
                const int column = first + 4 * lane;
                const bool mine = column < v_width && (VD != 96 || lane < 24);
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                if (mine) a = entries_of<LEAN>(p, at.row, p.v_from + column);
                const size_t to = ((size_t)at.page * p.num_v_heads + column / VD) * FRB_PAGE + at.in_page;
                store_codes<V_LANES>(a, mine, p.v_codes + to * VD + v_dim, p.v_scales + to, v_dim, p.codes);
            }
        t += gridDim.x;
        if (t >= p.num_tokens) return;
        tables();
        __syncthreads();                                    // the row is no longer needed
        if (threadIdx.x == 0) {
            const int next = t + (p.stages - 1) * (int)gridDim.x;
            if (next < p.num_tokens) ask(next, stage);
        }
    }
}

// Up to this many tokens (two for each of a B200's 148 SMs) a block has a warp for every two spans, up to 32; beyond, as many blocks as are resident take
// the tokens in turn.
#define WRITE8_FEW_TOKENS 296

FRB_API int frb_qkv_prepare_8bit(const void* qkv, int in_dtype, const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                                 const float* cos_table, const float* sin_table, int table_positions, const int* tok_pos,
                                 const int* tok_slot, const int* page_table, int num_slots, int max_pages, void* q_out, void* k_codes,
                                 float* k_scales, void* v_codes, float* v_scales, int codes, int num_pages, int num_tokens, int num_heads,
                                 int num_kv_heads, int num_v_heads, int head_dim, int v_dim, int rotary_dim, int interleaved, int per_head,
                                 int tables_final, const float* bias, float q_temp_coef, int q_temp_every, int values_from_keys, int* status,
                                 cudaStream_t stream) {
    if (num_tokens == 0) return 0;
    FRB_CHECK_ARG(num_tokens > 0 && num_heads > 0 && num_kv_heads > 0 && num_v_heads > 0 && num_kv_heads % num_v_heads == 0,
                  "qkv_prepare_8bit: %d tokens, %d heads, %d key heads over %d value heads", num_tokens, num_heads, num_kv_heads, num_v_heads);
    FRB_CHECK_ARG(codes == FRB_E4M3 || codes == FRB_INT8, "qkv_prepare_8bit: codes of type %d", codes);
    FRB_CHECK_ARG(!values_from_keys || (!k_weight && v_dim == head_dim && num_v_heads == num_kv_heads),
                  "qkv_prepare_8bit: values that are the keys as projected go without a norm of the keys and have the keys' heads and size");
    FRB_CHECK_ARG(q_temp_coef == 0.f || q_temp_every >= 1, "qkv_prepare_8bit: a query temperature every %d positions", q_temp_every);
    FRB_CHECK_ARG(rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim, "qkv_prepare_8bit: rotary_dim %d must be even and <= head_dim %d",
                  rotary_dim, head_dim);
    FRB_CHECK_ARG(rotary_dim == 0 || (cos_table && sin_table && table_positions > 0), "qkv_prepare_8bit: rotary tables are missing");
    const auto aligned = [](const void* ptr, uintptr_t bytes) { return ((uintptr_t)ptr & (bytes - 1)) == 0; };
    FRB_CHECK_ARG(aligned(qkv, 16) && aligned(bias, 16) && aligned(q_weight, weight_dtype == FRB_F32 ? 16 : 8) &&
                  aligned(k_weight, weight_dtype == FRB_F32 ? 16 : 8) && aligned(q_out, 8) && aligned(k_codes, 4) && aligned(v_codes, 4),
                  "qkv_prepare_8bit: rows start on 16 bytes, the other tensors on a whole group of four entries");
    Write8Params p;
    p.qkv = qkv; p.bias = bias; p.q_weight = q_weight; p.k_weight = k_weight; p.cos_table = cos_table; p.sin_table = sin_table;
    p.tok_pos = tok_pos; p.tok_slot = tok_slot; p.page_table = page_table; p.q_out = (bf16*)q_out; p.k_codes = (uint8_t*)k_codes;
    p.k_scales = k_scales; p.v_codes = (uint8_t*)v_codes; p.v_scales = v_scales; p.eps = eps; p.q_temp_coef = q_temp_coef;
    p.q_temp_every = q_temp_every > 0 ? q_temp_every : 1; p.num_heads = num_heads; p.num_kv_heads = num_kv_heads;
    p.num_v_heads = num_v_heads; p.rotary_dim = rotary_dim; p.interleaved = interleaved; p.max_pages = max_pages;
    p.num_slots = num_slots; p.num_pages = num_pages; p.table_positions = table_positions; p.per_head = per_head && (q_weight || k_weight);
    p.tables_final = tables_final; p.codes = codes; p.in_f32 = in_dtype == FRB_F32; p.weight_f32 = weight_dtype == FRB_F32;
    const long long width = (long long)(num_heads + num_kv_heads) * head_dim + (values_from_keys ? 0ll : (long long)num_v_heads * v_dim);
    FRB_CHECK_ARG(width <= (in_dtype == FRB_F32 ? 50000 : 100000), "qkv_prepare_8bit: a row of %lld entries needs more than 200 KB of shared memory", width);
    p.row_width = (int)width;
    p.v_from = (num_heads + (values_from_keys ? 0 : num_kv_heads)) * head_dim;
    const bool few = num_tokens <= WRITE8_FEW_TOKENS;
    const size_t row_bytes = (size_t)width * (in_dtype == FRB_F32 ? 4 : 2);
    const int spans = (int)((width + 127) / 128);
    // beyond a few tokens: a warp for every eight spans (what a warp does once per token is as much as a dozen spans), 24 warps an SM.  Rows of 16 KB and
    // more one at a time: with the next one's copy under way the blocks' shared memory would leave the L1 cache no room for the norms' weights.
    const int warps = few ? (spans < 2 ? 1 : spans > 64 ? 32 : spans / 2) : spans < 16 ? 2 : spans > 64 ? 8 : spans / 8;
    p.stages = few || row_bytes >= 16 * 1024 ? 1 : 2;
    const size_t smem = p.stages * row_bytes;
    int resident = (int)((p.stages == 1 ? 140 : 208) * 1024 / (smem + 1024));
    if (resident > 24 / warps) resident = 24 / warps;
    if (resident < 1) resident = 1;
    const long long most = few ? num_tokens : (long long)resident * frb_sm_count();
    const bool lean = in_dtype == FRB_F32 && weight_dtype == FRB_F32 && !bias;
    p.angles_by_four = aligned(cos_table, 16) && aligned(sin_table, 16);
    p.status = status;
    p.num_tokens = num_tokens;
#define FRB_LAUNCH_WRITE8(HD, VD)                                                                                                     \
    auto kernel = few ? (lean ? qkv_prepare_8bit_kernel<HD, VD, 1024, 1, true> : qkv_prepare_8bit_kernel<HD, VD, 1024, 1, false>)     \
                      : (lean ? qkv_prepare_8bit_kernel<HD, VD, 256, 3, true> : qkv_prepare_8bit_kernel<HD, VD, 256, 3, false>);      \
    if (smem > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);                       \
    launch_dependent(kernel, dim3((unsigned)(num_tokens < most ? num_tokens : most)), dim3(32 * warps), smem, stream, p)
    FRB_8BIT_SIZES("qkv_prepare_8bit", head_dim, v_dim, FRB_LAUNCH_WRITE8);
#undef FRB_LAUNCH_WRITE8
    FRB_RETURN_LAUNCH("qkv_prepare_8bit");
}

// ----------------------------------------------------------------------------- pages read back

struct Read8Params {
    const uint8_t* k_codes;   // [pages, nkv, 64, hd]
    const float* k_scales;
    const uint8_t* v_codes;   // [pages, nvh, 64, vd]
    const float* v_scales;
    const int* page_table;    // [slots, max_pages]
    const int* page_seq;      // [n] sequence (of the step) whose page this is
    const int* page_index;    // [n] number of the page in its sequence
    const int* seq_slot;      // [sequences]
    const int* seq_start;     // a sequence holds seq_start + seq_new tokens
    const int* seq_new;
    bf16* keys;               // [n, nkv, 64, hd]
    bf16* values;             // [n, nvh, vd, 64]
    int num_kv_heads, num_v_heads, num_pages, num_slots, max_pages, num_seqs, codes;
};

#define READ8_THREADS 256
#define READ8_CODES 2048       // codes that a warp takes at a time

// Two rounded to bfloat16.
__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A warp takes 2,048 codes of one head's page: a run of key rows, which go out as they came, or all 64 tokens of 32 dimensions of the
// values, which are turned on the way (the kernels that read them want a dimension's 64 tokens side by side).  For those a lane
// reads 16 dimensions of four neighbouring tokens and writes 16 times the four tokens of a dimension; the sixteen lanes with the same dimensions
// write a whole row of 128 bytes.  All of a lane's loads are under way before the first is used.  What bounds it is its bytes, one in and two
// out an entry.  Measured on a B200 with 512 pages of MiniMax-M2's heads (203 MB): 34 us, 5.9 TB/s.
// grid (page, share of its heads' 2,048 codes).
template <int HD, int VD, int CODES>
__global__ void __launch_bounds__(READ8_THREADS) cache_read_8bit_kernel(Read8Params p) {
    after_previous_kernel();
    constexpr int K_PARTS = HD / 32, V_PARTS = VD / 32;          // of a head's page
    const int n = blockIdx.x, lane = threadIdx.x & 31;
    const int part = blockIdx.y * (READ8_THREADS / 32) + (threadIdx.x >> 5), k_parts = p.num_kv_heads * K_PARTS;
    if (part >= k_parts + p.num_v_heads * V_PARTS) return;
    const int seq = p.page_seq[n], index = p.page_index[n];
    int page = -1, there = 0;                              // tokens of the page that the sequence holds
    if (seq >= 0 && seq < p.num_seqs && index >= 0 && index < p.max_pages) {
        const int slot = p.seq_slot[seq];
        if (slot >= 0 && slot < p.num_slots) page = p.page_table[(size_t)slot * p.max_pages + index];
        const long long left = (long long)p.seq_start[seq] + p.seq_new[seq] - (long long)index * FRB_PAGE;
        there = page >= 0 && page < p.num_pages ? (int)min(max(left, 0ll), (long long)FRB_PAGE) : 0;
    }
    page = there > 0 ? page : 0;
    if (part < k_parts) {
        const int head = part / K_PARTS, at = (part - head * K_PARTS) * READ8_CODES + 8 * lane;
        const size_t base = ((size_t)page * p.num_kv_heads + head) * FRB_PAGE;
        const uint8_t* codes = p.k_codes + base * HD;
        uint2 c[8];
        float s[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = at + 256 * u, token = i / HD;
            c[u] = token < there ? __ldg(reinterpret_cast<const uint2*>(codes + i)) : make_uint2(0u, 0u);
            s[u] = token < there ? __ldg(p.k_scales + base + token) : 0.f;
        }
        bf16* out = p.keys + ((size_t)n * p.num_kv_heads + head) * FRB_PAGE * HD;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float4 a = four_values(c[u].x, s[u], CODES), b = four_values(c[u].y, s[u], CODES);
            *reinterpret_cast<uint4*>(out + at + 256 * u) = make_uint4(two_bf16(a.x, a.y), two_bf16(a.z, a.w), two_bf16(b.x, b.y), two_bf16(b.z, b.w));
        }
    } else {
        const int at = part - k_parts, head = at / V_PARTS, dim = 32 * (at - head * V_PARTS) + 16 * (lane >> 4), token = 4 * (lane & 15);
        const size_t base = ((size_t)page * p.num_v_heads + head) * FRB_PAGE;
        const uint8_t* codes = p.v_codes + (base + token) * VD + dim;
        uint4 c[4];
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[i] = token + i < there ? __ldg(reinterpret_cast<const uint4*>(codes + (size_t)i * VD)) : make_uint4(0u, 0u, 0u, 0u);
            s[i] = token + i < there ? __ldg(p.v_scales + base + token + i) : 0.f;
        }
        bf16* out = p.values + (((size_t)n * p.num_v_heads + head) * VD + dim) * FRB_PAGE + token;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float4 v[4];                                   // [token][dimension]
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = four_values((&c[i].x)[w], s[i], CODES);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint2*>(out + (size_t)(4 * w + e) * FRB_PAGE) =
                    make_uint2(two_bf16((&v[0].x)[e], (&v[1].x)[e]), two_bf16((&v[2].x)[e], (&v[3].x)[e]));
        }
    }
}

FRB_API int frb_cache_read_8bit(const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales, int codes,
                                int num_pages, const int* page_table, int num_slots, int max_pages, const int* page_seq,
                                const int* page_index, int count, const int* seq_slot, const int* seq_start, const int* seq_new,
                                int num_seqs, void* keys, void* values, int num_kv_heads, int num_v_heads, int head_dim, int v_dim,
                                cudaStream_t stream) {
    if (count == 0) return 0;
    FRB_CHECK_ARG(count > 0 && num_kv_heads > 0 && num_v_heads > 0 && num_pages > 0 && num_slots > 0 && max_pages > 0 && num_seqs > 0,
                  "cache_read_8bit: %d pages of %d key heads and %d value heads", count, num_kv_heads, num_v_heads);
    FRB_CHECK_ARG(codes == FRB_E4M3 || codes == FRB_INT8, "cache_read_8bit: codes of type %d", codes);
    const auto aligned = [](const void* ptr, uintptr_t bytes) { return ((uintptr_t)ptr & (bytes - 1)) == 0; };
    FRB_CHECK_ARG(aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(keys, 16) && aligned(values, 16),
                  "cache_read_8bit: codes and pages start on 16 bytes");
    const int parts = num_kv_heads * (head_dim / 32) + num_v_heads * (v_dim / 32), shares = (parts + READ8_THREADS / 32 - 1) / (READ8_THREADS / 32);
    FRB_CHECK_ARG(num_kv_heads <= 65536 && num_v_heads <= 65536 && shares <= 65535, "cache_read_8bit: %d heads exceed the grid", num_kv_heads + num_v_heads);
    Read8Params p;
    p.k_codes = (const uint8_t*)k_codes; p.k_scales = k_scales; p.v_codes = (const uint8_t*)v_codes; p.v_scales = v_scales;
    p.page_table = page_table; p.page_seq = page_seq; p.page_index = page_index; p.seq_slot = seq_slot; p.seq_start = seq_start;
    p.seq_new = seq_new; p.keys = (bf16*)keys; p.values = (bf16*)values; p.num_kv_heads = num_kv_heads; p.num_v_heads = num_v_heads;
    p.num_pages = num_pages; p.num_slots = num_slots; p.max_pages = max_pages; p.num_seqs = num_seqs; p.codes = codes;
#define FRB_LAUNCH_READ8(HD, VD)                                                                                               \
    auto kernel = codes == FRB_E4M3 ? cache_read_8bit_kernel<HD, VD, FRB_E4M3> : cache_read_8bit_kernel<HD, VD, FRB_INT8>;     \
    launch_dependent(kernel, dim3(count, shares), dim3(READ8_THREADS), 0, stream, p)
    FRB_8BIT_SIZES("cache_read_8bit", head_dim, v_dim, FRB_LAUNCH_READ8);
#undef FRB_LAUNCH_READ8
    FRB_RETURN_LAUNCH("cache_read_8bit");
}

FRB_API int frb_qkv_prepare_8bit_packed(const void* packed, cudaStream_t stream) { return call_packed(frb_qkv_prepare_8bit, packed, stream); }

FRB_API int frb_cache_read_8bit_packed(const void* packed, cudaStream_t stream) { return call_packed(frb_cache_read_8bit, packed, stream); }
