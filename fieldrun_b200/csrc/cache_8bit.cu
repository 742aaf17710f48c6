// Rows written into a cache of 8-bit pages, and pages read back.
//
// qkv_prepare_8bit does what qkv_prepare does (bias, norms of queries and keys, rotation, the queries' temperature,
// src/minimax.rs:136-150, 253-268) and stores keys and values as codes with a scale a row (cache_8bit.cuh): the counterpart of
// the reference's row quantiser for its 8-bit cache (src/minimax.rs:291-347).  cache_read_8bit gives the rows of chosen pages
// back as bfloat16 pages in the layout that the prompt attention kernels read.
#include "cache_8bit.cuh"

using namespace frb_8bit;

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
    int per_head, tables_final, row_width, v_from, codes, in_f32, weight_f32;
};

__device__ __forceinline__ float4 four_of(const void* base, size_t at, int is_f32) {
    return is_f32 ? load4<float>(reinterpret_cast<const float*>(base) + at) : load4<bf16>(reinterpret_cast<const bf16*>(base) + at);
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

// The lane's part of a head's rotation: four dimensions from `dim` on.  Pairs of dimensions lie in the same four entries (interleaved), in two
// fours of neighbours (halves of a whole number of fours), or anywhere.
struct Turn {
    float4 cos, sin;           // of the lane's four dimensions; cos 1 and sin 0 where nothing turns
    int kind;                  // 0 none, 1 pairs of neighbours, 2 whole fours, 3 anywhere
    int from;                  // kind 2: the partners' lane

    template <int LANES>
    __device__ __forceinline__ void load(const Write8Params& p, int position, int dim, int lane) {
        cos = make_float4(1.f, 1.f, 1.f, 1.f);
        sin = make_float4(0.f, 0.f, 0.f, 0.f);
        const int rot = p.rotary_dim, half = rot / 2;
        kind = rot == 0 ? 0 : p.interleaved ? (rot % 4 == 0 ? 1 : 3) : rot % 8 == 0 ? 2 : 3;
        from = lane;
        if (rot == 0) return;
        const size_t row = (size_t)min(max(position, 0), p.table_positions - 1) * half;
        float* c = &cos.x;
        float* s = &sin.x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = dim + e;
            if (d >= rot) continue;
            const bool lower = p.interleaved ? (d & 1) == 0 : d < half;
            const int j = p.interleaved ? d >> 1 : lower ? d : d - half;
            c[e] = p.cos_table[row + j];
            // a' = a c - b s ; b' = b c + a s   (src/minimax.rs:78-81)
            s[e] = lower ? -p.sin_table[row + j] : p.sin_table[row + j];
        }
        if (kind == 2 && dim < rot) from = lane + (dim < half ? half / 4 : -half / 4);
    }

    template <int LANES>
    __device__ __forceinline__ float4 of(const Write8Params& p, float4 a, int dim, int lane) const {
        float4 b;
        if (kind == 0) return a;
        if (kind == 1) {
            b = make_float4(a.y, a.x, a.w, a.z);
        } else if (kind == 2) {
            b = make_float4(__shfl_sync(0xffffffffu, a.x, from), __shfl_sync(0xffffffffu, a.y, from), __shfl_sync(0xffffffffu, a.z, from),
                            __shfl_sync(0xffffffffu, a.w, from));
        } else {
            const int rot = p.rotary_dim, half = rot / 2;
            float r[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = dim + e, partner = d >= rot ? d : p.interleaved ? d ^ 1 : d < half ? d + half : d - half;
                const int at = (lane & ~(LANES - 1)) + (partner >> 2);
                const float x = __shfl_sync(0xffffffffu, a.x, at), y = __shfl_sync(0xffffffffu, a.y, at);
                const float z = __shfl_sync(0xffffffffu, a.z, at), w = __shfl_sync(0xffffffffu, a.w, at);
                r[e] = (partner & 2) == 0 ? ((partner & 1) == 0 ? x : y) : ((partner & 1) == 0 ? z : w);
            }
            b = make_float4(r[0], r[1], r[2], r[3]);
        }
        return make_float4(a.x * cos.x + b.x * sin.x, a.y * cos.y + b.y * sin.y, a.z * cos.z + b.z * sin.z, a.w * cos.w + b.w * sin.w);
    }
};

// One block per token, the row in registers: a warp takes spans of 32 lanes, four entries a lane (a head of 128, two of 64, four of 32; a head of
// 96 leaves eight lanes idle), up to SPANS of them, all asked for before the first is used.  A head's statistic, its largest entry and its
// pairs of dimensions are exchanges between lanes; only the statistics over whole rows go through shared memory.  What bounds it for
// prompts is the rows' bytes (4 an entry in, 2 a query entry and 1 a key or value entry out).  Measured on a B200 with MiniMax-M2's
// rows of 8,192 entries: WRITE
template <int HD, int VD, int SPANS, int THREADS>
__global__ void __launch_bounds__(THREADS) qkv_prepare_8bit_kernel(Write8Params p) {
    let_next_kernel_start();
    __shared__ float sums[2][THREADS / 32];
    constexpr int K_LANES = HD == 96 ? 32 : HD / 4, V_LANES = VD == 96 ? 32 : VD / 4;
    constexpr int K_HEADS = 32 / K_LANES, V_HEADS = 32 / V_LANES;              // heads of a span
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int q_width = p.num_heads * HD, qk_heads = p.num_heads + p.num_kv_heads;
    const int qk_spans = (qk_heads + K_HEADS - 1) / K_HEADS, spans = qk_spans + (p.num_v_heads + V_HEADS - 1) / V_HEADS;
    const int k_dim = 4 * (lane % K_LANES), v_dim = 4 * (lane % V_LANES);
    const float4 ones = make_float4(1.f, 1.f, 1.f, 1.f);
    int pos = 0, page = -1;
    Turn turn;
    // a position, slot or page that does not exist writes nothing
    const auto tables = [&] {
        pos = p.tok_pos[t];
        const int slot = p.tok_slot[t];
        if (pos >= 0 && pos / FRB_PAGE < p.max_pages && slot >= 0 && slot < p.num_slots)
            page = p.page_table[(size_t)slot * p.max_pages + pos / FRB_PAGE];
        if (page >= p.num_pages) page = -1;
        turn.load<K_LANES>(p, pos, k_dim, lane);
    };
    // positions, slots, pages and angles that were there before the kernel before this one began
    if (p.tables_final) tables();
    wait_for_previous_kernel();
    // the column that the lane's entries of a span begin at; -1 for a lane without any
    const auto column_of = [&](int span) {
        if (span < qk_spans) {
            const int head = span * K_HEADS + lane / K_LANES;
            return head < qk_heads && k_dim < HD ? head * HD + k_dim : -1;
        }
        const int head = (span - qk_spans) * V_HEADS + lane / V_LANES;
        return span < spans && head < p.num_v_heads && v_dim < VD ? p.v_from + head * VD + v_dim : -1;
    };
    float4 x[SPANS];
#pragma unroll
    for (int u = 0; u < SPANS; ++u) {
        const int column = column_of(warp + u * warps);
        x[u] = column >= 0 ? four_of(p.qkv, (size_t)t * p.row_width + column, p.in_f32) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (!p.tables_final) tables();
    if (p.bias) {
#pragma unroll
        for (int u = 0; u < SPANS; ++u) {
            const int column = column_of(warp + u * warps);
            if (column < 0) continue;
            const float4 b = *reinterpret_cast<const float4*>(p.bias + column);
            x[u] = make_float4(x[u].x + b.x, x[u].y + b.y, x[u].z + b.z, x[u].w + b.w);
        }
    }
    // statistics of whole rows
    float rinv_q = 1.f, rinv_k = 1.f;
    const bool whole = !p.per_head && p.q_weight;
    if (whole) {
        float ssq = 0.f, ssk = 0.f;
#pragma unroll
        for (int u = 0; u < SPANS; ++u) {
            const int span = warp + u * warps;
            if (span < qk_spans) {
                if (column_of(span) < q_width) ssq += squares(x[u]);          // (a lane without entries has zeros)
                else ssk += squares(x[u]);
            }
        }
        ssq = warp_sum(ssq);
        ssk = warp_sum(ssk);
        if (lane == 0) { sums[0][warp] = ssq; sums[1][warp] = ssk; }
        __syncthreads();
        ssq = warp_sum(lane < warps ? sums[0][lane] : 0.f);
        ssk = warp_sum(lane < warps ? sums[1][lane] : 0.f);
        rinv_q = 1.0f / sqrtf(ssq / (float)q_width + p.eps);
        rinv_k = 1.0f / sqrtf(ssk / (float)(p.num_kv_heads * HD) + p.eps);
    }
    const float q_temp = p.q_temp_coef == 0.f ? 1.f : 1.f + p.q_temp_coef * logf((float)((pos + 1) / p.q_temp_every) + 1.f);
    float4 head_wq = ones, head_wk = ones;                  // a norm per head has the same weights for every head
    if (p.per_head && k_dim < HD) {
        head_wq = four_of(p.q_weight, k_dim, p.weight_f32);
        head_wk = four_of(p.k_weight, k_dim, p.weight_f32);
    }
    const int in_page = pos & (FRB_PAGE - 1);
#pragma unroll
    for (int u = 0; u < SPANS; ++u) {
        const int span = warp + u * warps, column = column_of(span);
        float4 a = x[u];
        if (span < qk_spans) {
            const bool is_q = column < q_width;
            if (whole) {
                const float4 w = column < 0 ? ones : is_q ? four_of(p.q_weight, column, p.weight_f32) : four_of(p.k_weight, column - q_width, p.weight_f32);
                a = times(times(a, w), is_q ? rinv_q : rinv_k);
            } else if (p.per_head) {
                const float rinv = 1.0f / sqrtf(run_sum<K_LANES>(squares(a)) / (float)HD + p.eps);
                a = times(times(a, is_q ? head_wq : head_wk), rinv);
            }
            if (is_q) a = times(a, q_temp);
            a = turn.of<K_LANES>(p, a, k_dim, lane);
            if (is_q && column >= 0) store4<bf16>(p.q_out + (size_t)t * q_width + column, a);
            if ((span + 1) * K_HEADS > p.num_heads && page >= 0) {            // a key among the span's heads
                const uint32_t top = run_max<K_LANES>(largest(a));
                if (!is_q) {
                    float factor, scale;
                    row_scale(top, p.codes, factor, scale);
                    const int head = (column - q_width) / HD;
                    const size_t row = ((size_t)page * p.num_kv_heads + head) * FRB_PAGE + in_page;
                    *reinterpret_cast<uint32_t*>(p.k_codes + row * HD + k_dim) = four_codes(a, factor, p.codes);
                    if (k_dim == 0) p.k_scales[row] = scale;
                }
            }
        } else if (span < spans && page >= 0) {
            const uint32_t top = run_max<V_LANES>(largest(a));
            if (column >= 0) {
                float factor, scale;
                row_scale(top, p.codes, factor, scale);
                const int head = (column - p.v_from) / VD;
                const size_t row = ((size_t)page * p.num_v_heads + head) * FRB_PAGE + in_page;
                *reinterpret_cast<uint32_t*>(p.v_codes + row * VD + v_dim) = four_codes(a, factor, p.codes);
                if (v_dim == 0) p.v_scales[row] = scale;
            }
        }
    }
}

// Few tokens: two spans a warp, so that a token's loads are all under way at once on up to 32 warps; else eight (rows of up to 64 spans) or sixteen.
#define WRITE8_FEW_TOKENS 296

FRB_API int frb_qkv_prepare_8bit(const void* qkv, int in_dtype, const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                                 const float* cos_table, const float* sin_table, int table_positions, const int* tok_pos,
                                 const int* tok_slot, const int* page_table, int num_slots, int max_pages, void* q_out, void* k_codes,
                                 float* k_scales, void* v_codes, float* v_scales, int codes, int num_pages, int num_tokens, int num_heads,
                                 int num_kv_heads, int num_v_heads, int head_dim, int v_dim, int rotary_dim, int interleaved, int per_head,
                                 int tables_final, const float* bias, float q_temp_coef, int q_temp_every, int values_from_keys,
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
    FRB_CHECK_ARG(aligned(qkv, in_dtype == FRB_F32 ? 16 : 8) && aligned(bias, 16) && aligned(q_weight, weight_dtype == FRB_F32 ? 16 : 8) &&
                  aligned(k_weight, weight_dtype == FRB_F32 ? 16 : 8) && aligned(q_out, 8) && aligned(k_codes, 4) && aligned(v_codes, 4),
                  "qkv_prepare_8bit: a tensor does not start on a whole group of four entries");
    Write8Params p;
    p.qkv = qkv; p.bias = bias; p.q_weight = q_weight; p.k_weight = k_weight; p.cos_table = cos_table; p.sin_table = sin_table;
    p.tok_pos = tok_pos; p.tok_slot = tok_slot; p.page_table = page_table; p.q_out = (bf16*)q_out; p.k_codes = (uint8_t*)k_codes;
    p.k_scales = k_scales; p.v_codes = (uint8_t*)v_codes; p.v_scales = v_scales; p.eps = eps; p.q_temp_coef = q_temp_coef;
    p.q_temp_every = q_temp_every > 0 ? q_temp_every : 1; p.num_heads = num_heads; p.num_kv_heads = num_kv_heads;
    p.num_v_heads = num_v_heads; p.rotary_dim = rotary_dim; p.interleaved = interleaved; p.max_pages = max_pages;
    p.num_slots = num_slots; p.num_pages = num_pages; p.table_positions = table_positions; p.per_head = per_head && (q_weight || k_weight);
    p.tables_final = tables_final; p.codes = codes; p.in_f32 = in_dtype == FRB_F32; p.weight_f32 = weight_dtype == FRB_F32;
    const long long width = (long long)(num_heads + num_kv_heads) * head_dim + (values_from_keys ? 0ll : (long long)num_v_heads * v_dim);
    const int k_span = head_dim == 96 ? 1 : 128 / head_dim, v_span = v_dim == 96 ? 1 : 128 / v_dim;       // heads of a span
    const int spans = (num_heads + num_kv_heads + k_span - 1) / k_span + (num_v_heads + v_span - 1) / v_span;
    FRB_CHECK_ARG(num_heads <= 4096 && num_kv_heads <= 4096 && spans <= 256, "qkv_prepare_8bit: a row of %lld entries is more than 256 warps' loads", width);
    p.row_width = (int)width;
    p.v_from = (num_heads + (values_from_keys ? 0 : num_kv_heads)) * head_dim;
    const bool few = num_tokens <= WRITE8_FEW_TOKENS && spans <= 64;
    const int each = few ? 2 : spans <= 64 ? 8 : 16;
    const dim3 block(32 * ((spans + each - 1) / each));
#define FRB_LAUNCH_WRITE8(HD, VD)                                                                                                    \
    auto kernel = few ? qkv_prepare_8bit_kernel<HD, VD, 2, 1024> : spans <= 64 ? qkv_prepare_8bit_kernel<HD, VD, 8, 256>             \
                                                                               : qkv_prepare_8bit_kernel<HD, VD, 16, 512>;           \
    launch_dependent(kernel, dim3(num_tokens), block, 0, stream, p)
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
// out an entry.  Measured on a B200 with 512 pages of MiniMax-M2's heads (201 MB): READ
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
