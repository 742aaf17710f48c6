// The operators on 8-bit weights, each one call: a linear layer, a gated feed-forward block, routed experts.  The kernels are in
// rows_8bit.cu and products_8bit.cu; what passes between them lies in the caller's scratch.
#include "cache_8bit.cuh"          // call_packed
#include "products_8bit.cuh"

using namespace frb_products8;

// Runs of the scratch, each from a 256-byte boundary on.
struct Scratch {
    char* base;
    long long at = 0;
    explicit Scratch(void* p) : base((char*)p) {}
    template <typename T> T* take(long long count) {
        T* here = reinterpret_cast<T*>(base + at);
        at += (count * (long long)sizeof(T) + 255) / 256 * 256;
        return here;
    }
    bool starts_well() const { return ((uintptr_t)base & 15) == 0; }
};

// From one row of a unit's middle to the next: whole lines, whatever the width.
static int hidden_stride(int I) { return up_to(I, 32); }

#define FRB_TRY(call)                         \
    do {                                      \
        const int status_ = (call);           \
        if (status_ != 0) return status_;     \
    } while (0)

// Rows and the product that reads them: one launch where the product rounds them itself, else rows as codes in the scratch first.  The kernel
// that makes those lets the product start only after its own wait, so that the weights, whoever wrote them, are complete by then; before it where
// they are so anyway: behind another product (in_chain), which has waited so itself, and by the caller's word.
static int rows_and_product(Product& p, const void* x, int x_type, int x_stride, int8_t* codes, float* scales, bool weights_final, bool in_chain,
                            cudaStream_t stream) {
    if (!p.lists.tile_expert && tokens_fit(p.rows, p.K)) {
        p.x = x; p.x_type = x_type; p.x_stride = x_stride; p.x_scale = nullptr; p.weights_final = weights_final;
        return product(p, stream);
    }
    FRB_TRY(rows_codes(x, x_type, x_stride, p.rows, p.K, nullptr, 1, codes, scales, in_chain || weights_final, stream));
    p.x = codes; p.x_scale = scales; p.weights_final = true;
    return product(p, stream);
}

// out [T, F] = x [T, K] W^T; W as codes [F up to 16][K up to 128] with scales [F up to 16].  weights_final: they were complete before the kernel
// before this call began.  scratch: T (K up to 128) + 4 T bytes, each run up to 256, none where tokens_fit().
FRB_API int frb_linear_8bit(const void* x, int x_type, int T, int K, const void* w, const float* w_scale, int F, void* out, int out_type,
                            int weights_final, void* scratch, long long scratch_bytes, int* status, cudaStream_t stream) {
    if (T == 0) return 0;
    FRB_CHECK_ARG(K >= 1 && K <= FRB_8BIT_MOST_INNER, "linear in 8 bits: %d entries are outside 1..%d", K, FRB_8BIT_MOST_INNER);
    Scratch s(scratch);
    int8_t* codes = nullptr;
    float* scales = nullptr;
    if (!tokens_fit(T, K)) {
        codes = s.take<int8_t>((long long)T * up_to(K, FRB_8BIT_KBLOCK));
        scales = s.take<float>(T);
    }
    FRB_CHECK_ARG(s.at <= scratch_bytes, "linear in 8 bits: %lld bytes of scratch, %lld are needed", scratch_bytes, s.at);
    FRB_CHECK_ARG(s.starts_well(), "linear in 8 bits: the scratch starts on 16 bytes");
    const size_t x_bytes = (size_t)T * K * (x_type == FRB_F32 ? 4 : 2), out_bytes = (size_t)T * F * (out_type == FRB_F32 ? 4 : 2);
    FRB_CHECK_ARG((uintptr_t)x + x_bytes <= (uintptr_t)out || (uintptr_t)out + out_bytes <= (uintptr_t)x,
                  "linear in 8 bits: the results lie on the rows that they are made of");
    Product p = {};
    p.w = w; p.w_scale = w_scale; p.experts = 1; p.parts = 1; p.F = F; p.K = K; p.rows = T; p.out = out; p.out_stride = F; p.out_type = out_type;
    p.status = status;
    return rows_and_product(p, x, x_type, K, codes, scales, weights_final != 0, false, stream);
}

// h = act(x Wg^T) * (x Wu^T) in float32, rounded to codes row by row, out [T, d] = h Wd^T.  w_in: codes [2][I up to 16][d up to 128] (gate, up),
// w_down: [d up to 16][I up to 128].
FRB_API int frb_gated_8bit(const void* x, int x_type, int T, int d, const void* w_in, const float* in_scale, int I, const void* w_down,
                           const float* down_scale, int gate, float limit, void* out, int out_type, int weights_final, void* scratch,
                           long long scratch_bytes, int* status, cudaStream_t stream) {
    if (T == 0) return 0;
    FRB_CHECK_ARG(d >= 1 && d <= FRB_8BIT_MOST_INNER && I >= 1 && I <= FRB_8BIT_MOST_INNER, "gated block in 8 bits: %d entries, %d between, outside 1..%d", d, I,
                  FRB_8BIT_MOST_INNER);
    FRB_CHECK_ARG(gate == FRB_GATE_SILU || gate == FRB_GATE_GELU_TANH, "gated block in 8 bits: activation %d", gate);
    Scratch s(scratch);
    int8_t* codes = s.take<int8_t>((long long)T * up_to(d, FRB_8BIT_KBLOCK));
    float* scales = s.take<float>(T);
    const int IP = hidden_stride(I);
    float* hidden = s.take<float>((long long)T * IP);
    int8_t* hidden_codes = s.take<int8_t>((long long)T * up_to(I, FRB_8BIT_KBLOCK));
    float* hidden_scales = s.take<float>(T);
    FRB_CHECK_ARG(s.at <= scratch_bytes, "gated block in 8 bits: %lld bytes of scratch, %lld are needed", scratch_bytes, s.at);
    FRB_CHECK_ARG(s.starts_well(), "gated block in 8 bits: the scratch starts on 16 bytes");
    Product p = {};
    p.w = w_in; p.w_scale = in_scale; p.experts = 1; p.parts = 2; p.F = I; p.K = d; p.rows = T; p.out = hidden; p.out_stride = IP;
    p.out_type = FRB_F32; p.gate = gate; p.limit = limit; p.status = status;
    FRB_TRY(rows_and_product(p, x, x_type, d, codes, scales, weights_final != 0, false, stream));
    p.w = w_down; p.w_scale = down_scale; p.parts = 1; p.F = d; p.K = I; p.out = out; p.out_stride = d; p.out_type = out_type;
    return rows_and_product(p, hidden, FRB_F32, IP, hidden_codes, hidden_scales, true, true, stream);
}

// The experts' outputs y [N, d] (float32, rows y_stride apart, in the order of the lists) for T tokens that were given their rows already: row_of_assign
// [T, top_k], or null where x holds the rows in that order (top_k 1).
static int expert_rows(const void* x, int x_type, int T, int d, int top_k, const int* row_of_assign, const Lists& lists, const void* w_in,
                       const float* in_scale, int experts, int I, const void* w_down, const float* down_scale, float limit, float* y, int y_stride,
                       Scratch& s, long long scratch_bytes, int* status, cudaStream_t stream) {
    FRB_CHECK_ARG(row_of_assign != nullptr || top_k == 1, "experts in 8 bits: rows in order go to one expert each, not %d", top_k);
    const int N = T * top_k;
    int8_t* codes = s.take<int8_t>((long long)N * up_to(d, FRB_8BIT_KBLOCK));
    float* scales = s.take<float>(N);
    const int IP = hidden_stride(I);
    float* hidden = s.take<float>((long long)N * IP);
    int8_t* hidden_codes = s.take<int8_t>((long long)N * up_to(I, FRB_8BIT_KBLOCK));
    float* hidden_scales = s.take<float>(N);
    FRB_CHECK_ARG(s.at <= scratch_bytes, "experts in 8 bits: %lld bytes of scratch, %lld are needed", scratch_bytes, s.at);
    FRB_CHECK_ARG(s.starts_well(), "experts in 8 bits: the scratch starts on 16 bytes");
    FRB_TRY(rows_codes(x, x_type, d, T, d, row_of_assign, top_k, codes, scales, false, stream));
    Product p = {};
    p.w = w_in; p.w_scale = in_scale; p.experts = experts; p.parts = 2; p.F = I; p.K = d; p.rows = N; p.x = codes; p.x_scale = scales;
    p.lists = lists;
    p.out = hidden; p.out_stride = IP; p.out_type = FRB_F32; p.gate = FRB_GATE_SILU; p.limit = limit; p.status = status; p.weights_final = true;
    FRB_TRY(product(p, stream));
    FRB_TRY(rows_codes(hidden, FRB_F32, IP, N, I, nullptr, 1, hidden_codes, hidden_scales, true, stream));
    p.w = w_down; p.w_scale = down_scale; p.parts = 1; p.F = d; p.K = I; p.x = hidden_codes; p.x_scale = hidden_scales; p.out = y; p.out_stride = y_stride;
    return product(p, stream);
}

// The same with one row behind another.
FRB_API int frb_expert_rows_8bit(const void* x, int x_type, int T, int d, int top_k, const int* row_of_assign, const int* tile_expert, const int* tile_row0,
                                 const int* num_tiles, const int* offsets, int max_tiles, int tile_rows, const void* w_in, const float* in_scale, int experts,
                                 int I, const void* w_down, const float* down_scale, float limit, float* y, void* scratch, long long scratch_bytes, int* status,
                                 cudaStream_t stream) {
    if (T == 0) return 0;
    FRB_CHECK_ARG((long long)T * top_k < (1ll << 30), "experts in 8 bits: %d tokens of %d experts", T, top_k);
    Scratch s(scratch);
    return expert_rows(x, x_type, T, d, top_k, row_of_assign, {tile_expert, tile_row0, num_tiles, offsets, max_tiles, tile_rows}, w_in, in_scale, experts, I,
                       w_down, down_scale, limit, y, d, s, scratch_bytes, status, stream);
}

// out [T, d] = sum over r of weights[t, r] * unit of expert ids[t, r] on x[t].  w_in: codes [experts][2][I up to 16][d up to 128], w_down:
// [experts][d up to 16][I up to 128].
FRB_API int frb_experts_8bit(const void* x, int x_type, int T, int d, int top_k, const int* ids, const float* weights, const void* w_in,
                             const float* in_scale, int experts, int I, const void* w_down, const float* down_scale, float limit, int tile_rows, void* out,
                             int out_type, void* scratch, long long scratch_bytes, int* status, cudaStream_t stream) {
    if (T == 0) return 0;
    FRB_CHECK_ARG((long long)T * top_k < (1ll << 30), "experts in 8 bits: %d tokens of %d experts", T, top_k);
    FRB_CHECK_ARG(experts >= 1 && experts <= 8192, "experts in 8 bits: %d experts are outside 1..8192", experts);
    FRB_CHECK_ARG(tile_rows >= 1, "experts in 8 bits: tiles of %d rows", tile_rows);
    const int N = T * top_k, max_tiles = N / tile_rows + (experts < N ? experts : N);
    Scratch s(scratch);
    int* offsets = s.take<int>(experts + 1);
    int* row_of_assign = s.take<int>(N);
    int* tile_expert = s.take<int>(max_tiles);
    int* tile_row0 = s.take<int>(max_tiles);
    int* num_tiles = s.take<int>(1);
    const int y_stride = hidden_stride(d);
    float* y = s.take<float>((long long)N * y_stride);
    FRB_CHECK_ARG(s.at <= scratch_bytes, "experts in 8 bits: %lld bytes of scratch, more are needed", scratch_bytes);
    FRB_CHECK_ARG(s.starts_well(), "experts in 8 bits: the scratch starts on 16 bytes");       // (the lists, too, are written into it)
    FRB_TRY(plan(ids, T, top_k, experts, tile_rows, offsets, row_of_assign, tile_expert, tile_row0, num_tiles, stream));
    FRB_TRY(expert_rows(x, x_type, T, d, top_k, row_of_assign, {tile_expert, tile_row0, num_tiles, offsets, max_tiles, tile_rows}, w_in, in_scale, experts, I,
                        w_down, down_scale, limit, y, y_stride, s, scratch_bytes, status, stream));
    return combine(y, y_stride, weights, row_of_assign, T, top_k, d, out, out_type, stream);
}

FRB_API int frb_linear_8bit_packed(const void* packed, cudaStream_t stream) { return call_packed(frb_linear_8bit, packed, stream); }
FRB_API int frb_gated_8bit_packed(const void* packed, cudaStream_t stream) { return call_packed(frb_gated_8bit, packed, stream); }
FRB_API int frb_expert_rows_8bit_packed(const void* packed, cudaStream_t stream) { return call_packed(frb_expert_rows_8bit, packed, stream); }
FRB_API int frb_experts_8bit_packed(const void* packed, cudaStream_t stream) { return call_packed(frb_experts_8bit, packed, stream); }
