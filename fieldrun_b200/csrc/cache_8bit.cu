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

// The largest of `v` over runs of LANES lanes.
template <int LANES>
__device__ __forceinline__ uint32_t run_max(uint32_t v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <int LANES>
__device__ __forceinline__ float run_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}


// One block per token.  The row comes into shared memory with the norms' weights multiplied in (all loads of a thread before their
// first use) while the sums of squares are taken; then a run of lanes takes a head, four entries a lane (32 lanes for heads of 96 and
// 128, 16 for 64, 8 for 32), so that a head's statistic and its largest entry are a few exchanges between lanes and a row of
// codes is one store.
template <int HD, int VD, int BLOCK>
__global__ void __launch_bounds__(BLOCK) qkv_prepare_8bit_kernel(Write8Params p) {
    let_next_kernel_start();
    extern __shared__ __align__(16) float raw[];   // the row, weighted; then cos and sin [rotary_dim / 2]
    __shared__ float scratch[64];
    constexpr int BATCH = BLOCK == 1024 ? 2 : 4;   // groups of four entries a thread loads before it uses any of them
    constexpr int K_LANES = HD == 96 ? 32 : HD / 4, V_LANES = VD == 96 ? 32 : VD / 4;
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int q_width = p.num_heads * HD, k_width = p.num_kv_heads * HD, qk_width = q_width + k_width;
    const int half = p.rotary_dim / 2;
    float* s_cos = raw + p.row_width;
    float* s_sin = s_cos + half;
    int pos = 0, page = -1;
    // a position, slot or page that does not exist writes nothing
    const auto tables = [&] {
        pos = p.tok_pos[t];
        const int slot = p.tok_slot[t];
        const int row = min(max(pos, 0), p.table_positions - 1);
        for (int j = threadIdx.x; j < half; j += BLOCK) {
            s_cos[j] = p.cos_table[(size_t)row * half + j];
            s_sin[j] = p.sin_table[(size_t)row * half + j];
        }
        if (pos >= 0 && pos / FRB_PAGE < p.max_pages && slot >= 0 && slot < p.num_slots)
            page = p.page_table[(size_t)slot * p.max_pages + pos / FRB_PAGE];
        if (page >= p.num_pages) page = -1;
    };
    // positions, slots, pages and angles that were there before the kernel before this one began
    if (p.tables_final) tables();
    wait_for_previous_kernel();
    if (!p.tables_final) tables();

    // a norm per head has the same weights for every head: a lane's four entries of them
    float4 head_wq = make_float4(1.f, 1.f, 1.f, 1.f), head_wk = head_wq;
    if (p.per_head && 4 * (lane % K_LANES) < HD) {
        if (p.q_weight) head_wq = four_of(p.q_weight, 4 * (lane % K_LANES), p.weight_f32);
        if (p.k_weight) head_wk = four_of(p.k_weight, 4 * (lane % K_LANES), p.weight_f32);
    }
    float ssq = 0.f, ssk = 0.f;
    for (int base = 0; base < p.row_width; base += 4 * BATCH * BLOCK) {
        float4 v[BATCH], w[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const int i = base + 4 * (u * BLOCK + threadIdx.x);
            v[u] = i < p.row_width ? four_of(p.qkv, (size_t)t * p.row_width + i, p.in_f32) : make_float4(0.f, 0.f, 0.f, 0.f);
            if (p.bias && i < p.row_width) {
                const float4 b = *reinterpret_cast<const float4*>(p.bias + i);
                v[u] = make_float4(v[u].x + b.x, v[u].y + b.y, v[u].z + b.z, v[u].w + b.w);
            }
            w[u] = make_float4(1.f, 1.f, 1.f, 1.f);
            if (p.per_head) continue;
            if (i < q_width) { if (p.q_weight) w[u] = four_of(p.q_weight, i, p.weight_f32); }
            else if (i < qk_width) { if (p.k_weight) w[u] = four_of(p.k_weight, i - q_width, p.weight_f32); }
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const int i = base + 4 * (u * BLOCK + threadIdx.x);
            if (i < p.row_width)
                *reinterpret_cast<float4*>(raw + i) = make_float4(v[u].x * w[u].x, v[u].y * w[u].y, v[u].z * w[u].z, v[u].w * w[u].w);
            const float ss = v[u].x * v[u].x + v[u].y * v[u].y + v[u].z * v[u].z + v[u].w * v[u].w;
            if (i < q_width) ssq += ss;
            else if (i < qk_width) ssk += ss;
        }
    }
    float rinv_q = 1.f, rinv_k = 1.f;
    if (!p.per_head && (p.q_weight || p.k_weight)) {
        block_sum_pair<BLOCK>(ssq, ssk, scratch);
        if (p.q_weight) rinv_q = 1.0f / sqrtf(ssq / (float)q_width + p.eps);
        if (p.k_weight) rinv_k = 1.0f / sqrtf(ssk / (float)k_width + p.eps);
    } else {
        __syncthreads();
    }
    if (p.q_temp_coef != 0.f) rinv_q *= 1.f + p.q_temp_coef * logf((float)((pos + 1) / p.q_temp_every) + 1.f);

    // queries and keys, a head to a run of lanes
    const int in_page = pos & (FRB_PAGE - 1);
    constexpr int K_RUNS = 32 / K_LANES, V_RUNS = 32 / V_LANES;
    const int qk_heads = p.num_heads + p.num_kv_heads;
    for (int first = warp * K_RUNS; first < qk_heads; first += BLOCK / 32 * K_RUNS) {
        const int head = first + lane / K_LANES, dim = 4 * (lane % K_LANES);
        const bool mine = head < qk_heads && dim < HD, is_q = head < p.num_heads;
        float* base = raw + (size_t)min(head, qk_heads - 1) * HD;
        float4 a = mine ? *reinterpret_cast<const float4*>(base + dim) : make_float4(0.f, 0.f, 0.f, 0.f);
        float rinv = is_q ? rinv_q : rinv_k;
        if (p.per_head) {
            const float ss = run_sum<K_LANES>(a.x * a.x + a.y * a.y + a.z * a.z + a.w * a.w);
            if (is_q ? p.q_weight != nullptr : p.k_weight != nullptr) {
                rinv *= 1.0f / sqrtf(ss / (float)HD + p.eps);
                const float4 w = is_q ? head_wq : head_wk;
                a = make_float4(a.x * w.x, a.y * w.y, a.z * w.z, a.w * w.w);
                if (mine) *reinterpret_cast<float4*>(base + dim) = a;        // for the lanes whose partners these are
            }
            __syncwarp();
        }
        a = make_float4(a.x * rinv, a.y * rinv, a.z * rinv, a.w * rinv);
        if (mine && dim < p.rotary_dim) {
            // a' = a c - b s ; b' = b c + a s   (src/minimax.rs:78-81)
            if (p.interleaved && p.rotary_dim % 4 == 0) {
                const int j = dim >> 1;
                const float c0 = s_cos[j], s0 = s_sin[j], c1 = s_cos[j + 1], s1 = s_sin[j + 1];
                a = make_float4(a.x * c0 - a.y * s0, a.y * c0 + a.x * s0, a.z * c1 - a.w * s1, a.w * c1 + a.z * s1);
            } else if (!p.interleaved && p.rotary_dim % 8 == 0) {
                const bool lower = dim < half;
                const int j = lower ? dim : dim - half;
                float4 b = *reinterpret_cast<const float4*>(base + (lower ? dim + half : dim - half));
                b = make_float4(b.x * rinv, b.y * rinv, b.z * rinv, b.w * rinv);
                const float c[4] = {s_cos[j], s_cos[j + 1], s_cos[j + 2], s_cos[j + 3]};
                const float n[4] = {s_sin[j], s_sin[j + 1], s_sin[j + 2], s_sin[j + 3]};
                if (lower) a = make_float4(a.x * c[0] - b.x * n[0], a.y * c[1] - b.y * n[1], a.z * c[2] - b.z * n[2], a.w * c[3] - b.w * n[3]);
                else a = make_float4(a.x * c[0] + b.x * n[0], a.y * c[1] + b.y * n[1], a.z * c[2] + b.z * n[2], a.w * c[3] + b.w * n[3]);
            } else {                                  // a pair may lie in two groups of four, or the rotation end inside one
                float r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = dim + e;
                    if (d >= p.rotary_dim) continue;
                    const bool lower = p.interleaved ? (d & 1) == 0 : d < half;
                    const int j = p.interleaved ? d >> 1 : lower ? d : d - half;
                    const int partner = p.interleaved ? d ^ 1 : lower ? d + half : d - half;
                    const float other = base[partner] * rinv;
                    r[e] = lower ? r[e] * s_cos[j] - other * s_sin[j] : r[e] * s_cos[j] + other * s_sin[j];
                }
                a = make_float4(r[0], r[1], r[2], r[3]);
            }
        }
        if (mine && is_q) store4<bf16>(p.q_out + (size_t)t * q_width + (size_t)head * HD + dim, a);
        const uint32_t top = run_max<K_LANES>(max(max(magnitude_bits(a.x), magnitude_bits(a.y)), max(magnitude_bits(a.z), magnitude_bits(a.w))));
        if (mine && !is_q && page >= 0) {
            float factor, scale;
            row_scale(top, p.codes, factor, scale);
            const size_t row = ((size_t)page * p.num_kv_heads + (head - p.num_heads)) * FRB_PAGE + in_page;
            *reinterpret_cast<uint32_t*>(p.k_codes + row * HD + dim) = four_codes(a, factor, p.codes);
            if (dim == 0) p.k_scales[row] = scale;
        }
    }
    for (int first = warp * V_RUNS; first < p.num_v_heads; first += BLOCK / 32 * V_RUNS) {
        const int head = first + lane / V_LANES, dim = 4 * (lane % V_LANES);
        const bool mine = head < p.num_v_heads && dim < VD;
        const float4 a = mine ? *reinterpret_cast<const float4*>(raw + p.v_from + (size_t)head * VD + dim) : make_float4(0.f, 0.f, 0.f, 0.f);
        const uint32_t top = run_max<V_LANES>(max(max(magnitude_bits(a.x), magnitude_bits(a.y)), max(magnitude_bits(a.z), magnitude_bits(a.w))));
        if (mine && page >= 0) {
            float factor, scale;
            row_scale(top, p.codes, factor, scale);
            const size_t row = ((size_t)page * p.num_v_heads + head) * FRB_PAGE + in_page;
            *reinterpret_cast<uint32_t*>(p.v_codes + row * VD + dim) = four_codes(a, factor, p.codes);
            if (dim == 0) p.v_scales[row] = scale;
        }
    }
}

#define WRITE8_FEW_TOKENS 296        // up to this many tokens a block has 1024 threads, else 256

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
    const size_t smem = ((size_t)width + rotary_dim) * sizeof(float);
    FRB_CHECK_ARG(width < (1 << 24) && smem <= 200 * 1024, "qkv_prepare_8bit: a row of %lld entries needs more than 200 KB of shared memory", width);
    p.row_width = (int)width;
    p.v_from = (num_heads + (values_from_keys ? 0 : num_kv_heads)) * head_dim;
#define FRB_LAUNCH_WRITE8(HD, VD)                                                                                                    \
    auto kernel = num_tokens <= WRITE8_FEW_TOKENS ? qkv_prepare_8bit_kernel<HD, VD, 1024> : qkv_prepare_8bit_kernel<HD, VD, 256>;    \
    if (smem > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);                      \
    launch_dependent(kernel, dim3(num_tokens), dim3(num_tokens <= WRITE8_FEW_TOKENS ? 1024 : 256), smem, stream, p)
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

// Block (page, head): the key heads of a page, then its value heads.  A key row goes out as it came; a page of values is turned in shared
// memory, because the kernels that read it want a dimension's 64 tokens side by side.
template <int HD, int VD>
__global__ void __launch_bounds__(READ8_THREADS) cache_read_8bit_kernel(Read8Params p) {
    after_previous_kernel();
    const int heads = p.num_kv_heads + p.num_v_heads;
    const int n = blockIdx.x / heads, h = blockIdx.x - n * heads;
    const bool is_key = h < p.num_kv_heads;
    const int seq = p.page_seq[n], index = p.page_index[n];
    int page = -1, there = 0;                              // tokens of the page that the sequence holds
    if (seq >= 0 && seq < p.num_seqs && index >= 0 && index < p.max_pages) {
        const int slot = p.seq_slot[seq];
        if (slot >= 0 && slot < p.num_slots) page = p.page_table[(size_t)slot * p.max_pages + index];
        const long long left = (long long)p.seq_start[seq] + p.seq_new[seq] - (long long)index * FRB_PAGE;
        there = page >= 0 && page < p.num_pages ? (int)min(max(left, 0ll), (long long)FRB_PAGE) : 0;
    }
    if (is_key) {
        const uint8_t* codes = p.k_codes + ((size_t)max(page, 0) * p.num_kv_heads + h) * FRB_PAGE * HD;
        const float* scales = p.k_scales + ((size_t)max(page, 0) * p.num_kv_heads + h) * FRB_PAGE;
        bf16* out = p.keys + ((size_t)n * p.num_kv_heads + h) * FRB_PAGE * HD;
        for (int i = 4 * threadIdx.x; i < FRB_PAGE * HD; i += 4 * READ8_THREADS) {
            const int token = i / HD;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (token < there) x = four_values(*reinterpret_cast<const uint32_t*>(codes + i), scales[token], p.codes);
            store4<bf16>(out + i, x);
        }
    } else {
        __shared__ bf16 tile[VD][FRB_PAGE + 2];
        const int vh = h - p.num_kv_heads;
        const uint8_t* codes = p.v_codes + ((size_t)max(page, 0) * p.num_v_heads + vh) * FRB_PAGE * VD;
        const float* scales = p.v_scales + ((size_t)max(page, 0) * p.num_v_heads + vh) * FRB_PAGE;
        bf16* out = p.values + ((size_t)n * p.num_v_heads + vh) * FRB_PAGE * VD;
        for (int i = 4 * threadIdx.x; i < FRB_PAGE * VD; i += 4 * READ8_THREADS) {
            const int token = i / VD, dim = i - token * VD;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (token < there) x = four_values(*reinterpret_cast<const uint32_t*>(codes + i), scales[token], p.codes);
            tile[dim][token] = __float2bfloat16_rn(x.x); tile[dim + 1][token] = __float2bfloat16_rn(x.y);
            tile[dim + 2][token] = __float2bfloat16_rn(x.z); tile[dim + 3][token] = __float2bfloat16_rn(x.w);
        }
        __syncthreads();
        for (int i = 2 * threadIdx.x; i < FRB_PAGE * VD; i += 2 * READ8_THREADS) {
            const int dim = i / FRB_PAGE, token = i - dim * FRB_PAGE;
            *reinterpret_cast<uint32_t*>(out + i) = *reinterpret_cast<const uint32_t*>(&tile[dim][token]);
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
    const long long blocks = (long long)count * (num_kv_heads + num_v_heads);
    FRB_CHECK_ARG(blocks < (1ll << 31), "cache_read_8bit: %d pages of %d heads exceed the grid", count, num_kv_heads + num_v_heads);
    Read8Params p;
    p.k_codes = (const uint8_t*)k_codes; p.k_scales = k_scales; p.v_codes = (const uint8_t*)v_codes; p.v_scales = v_scales;
    p.page_table = page_table; p.page_seq = page_seq; p.page_index = page_index; p.seq_slot = seq_slot; p.seq_start = seq_start;
    p.seq_new = seq_new; p.keys = (bf16*)keys; p.values = (bf16*)values; p.num_kv_heads = num_kv_heads; p.num_v_heads = num_v_heads;
    p.num_pages = num_pages; p.num_slots = num_slots; p.max_pages = max_pages; p.num_seqs = num_seqs; p.codes = codes;
#define FRB_LAUNCH_READ8(HD, VD) launch_dependent(cache_read_8bit_kernel<HD, VD>, dim3((unsigned)blocks), dim3(READ8_THREADS), 0, stream, p)
    FRB_8BIT_SIZES("cache_read_8bit", head_dim, v_dim, FRB_LAUNCH_READ8);
#undef FRB_LAUNCH_READ8
    FRB_RETURN_LAUNCH("cache_read_8bit");
}
