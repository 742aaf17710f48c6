// Rows as 8-bit codes with a scale, and what routed experts need around their products: lists of each expert's rows, and the sum over
// a token's experts.
#include "products_8bit.cuh"

namespace frb_products8 {

// ----------------------------------------------------------------------------- rows as codes

// Runs of 8 entries that a thread keeps in registers; what is beyond is read a second time (from L1).  512 threads a row are for few rows: one run
// each, and code that is short, since it comes cold (200 rows of 4,096 bfloat16: 3.4 us with four, 2.2 with one).  They also take the rows that are too
// long for 256 threads' registers, however many there are; of these all entries behind the first 4,096 are read twice.
constexpr int kept_runs(int per_row) { return per_row == 512 ? 1 : 4; }

// A row is taken by PER_ROW threads, a block of 128 or more holds one or several.  Bound by memory where there are many rows (2,048 of 8192
// float32 by 512 threads each 24 us, by 256 with all of their entries in registers 16), by two trips to it and the row's maximum where there
// are few.  `places`: row t goes to the rows places[t * copies + c] of the result (nowhere where that is none of them),
// else to row t.
template <typename T, int PER_ROW>
__global__ void __launch_bounds__(PER_ROW < 128 ? 128 : PER_ROW, PER_ROW == 512 ? 2 : (sizeof(T) == 4 ? 6 : 8) / (PER_ROW == 256 ? 2 : 1))
rows_8bit_kernel(const T* __restrict__ x, int x_stride, int rows, int K, int KP, const int* __restrict__ places, int copies, int places_end, int8_t* __restrict__ codes,
                 float* __restrict__ scales, int whole_rows, int early) {
    constexpr int BLOCK = PER_ROW < 128 ? 128 : PER_ROW, AT_ONCE = BLOCK / PER_ROW, KEPT = kept_runs(PER_ROW);
    __shared__ uint32_t warp_top[2][BLOCK / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, me = threadIdx.x % PER_ROW;
    // The kernel after this one may read ahead what kernels before this one wrote, so it starts after the wait; before it (early) where
    // that is complete already, so that a product has its first weights when this one ends (between two products 2.5 us of 117).
    if (early) let_next_kernel_start();
    wait_for_previous_kernel();
    if (!early) let_next_kernel_start();
    int turn = 0;
    for (int base = blockIdx.x * AT_ONCE; base < rows; base += gridDim.x * AT_ONCE, turn ^= 1) {
        const int row = base + threadIdx.x / PER_ROW;
        const bool there = AT_ONCE == 1 || row < rows;          // (a block's last rows may be none; its barrier is for all)
        const T* src = x + (size_t)(there ? row : 0) * x_stride;
        Eight<T> kept[KEPT];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < KEPT; ++j) {
            const int k = (j * PER_ROW + me) * 8;
            if (k < K) kept[j].read(src + k, K - k, whole_rows);
            else kept[j].clear();
        }
#pragma unroll
        for (int j = 0; j < KEPT; ++j) top = top_of(kept[j], top);
        for (int k = (KEPT * PER_ROW + me) * 8; k < K; k += PER_ROW * 8) {
            Eight<T> v;
            v.read(src + k, K - k, whole_rows);
            top = top_of(v, top);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (PER_ROW > 32) {
            if (lane == 0) warp_top[turn][warp] = top;
            __syncthreads();           // (two sets of maxima in turn: a warp that is ahead writes the other)
            constexpr int WARPS = PER_ROW / 32;                   // of a row
            top = __reduce_max_sync(0xffffffffu, lane < WARPS ? warp_top[turn][warp / WARPS * WARPS + lane] : 0u);
        }
        if (!there) continue;
        const float a = __uint_as_float(top);
        float factor, scale;
        row_factor<T>(top, factor, scale);
        uint2 made[KEPT];
        uint32_t again = 0;            // one bit for each run of eight entries that slow_codes() decides
#pragma unroll
        for (int j = 0; j < KEPT; ++j) {
            bool near;
            made[j] = codes_of(kept[j], factor, near);
            again |= (uint32_t)near << j;
        }
        const int count = places ? copies : 1;
#pragma unroll 1
        for (int i = 0; i < count; ++i) {
            const int to = places ? places[(size_t)row * copies + i] : row;
            if ((unsigned)to >= (unsigned)places_end) continue;
            int8_t* dst = codes + (size_t)to * KP;
#pragma unroll
            for (int j = 0; j < KEPT; ++j) {
                const int k = (j * PER_ROW + me) * 8;
                if (k < KP) *reinterpret_cast<uint2*>(dst + k) = made[j];
            }
            if (me == 0) scales[to] = scale;
        }
        const auto put = [&](int k, uint2 c) {
#pragma unroll 1
            for (int i = 0; i < count; ++i) {
                const int to = places ? places[(size_t)row * copies + i] : row;
                if ((unsigned)to < (unsigned)places_end) *reinterpret_cast<uint2*>(codes + (size_t)to * KP + k) = c;
            }
        };
#pragma unroll 1
        for (int j = 0; again >> j; ++j) {
            const int k = (j * PER_ROW + me) * 8;
            if ((again >> j & 1) && k < K) put(k, slow_codes(src + k, K - k, factor, a));
        }
#pragma unroll 1
        for (int k = (KEPT * PER_ROW + me) * 8; k < KP; k += PER_ROW * 8) {
            Eight<T> v;
            if (k < K) v.read(src + k, K - k, whole_rows);
            else v.clear();
            bool near;
            const uint2 c = codes_of(v, factor, near);
            put(k, near ? slow_codes(src + k, K - k, factor, a) : c);
        }
    }
}

int rows_codes(const void* x, int x_type, int x_stride, int rows, int K, const int* places, int copies, void* codes, float* scales, bool early, cudaStream_t stream) {
    if (rows == 0) return 0;
    FRB_CHECK_ARG(K >= 1 && K <= FRB_8BIT_MOST_INNER, "rows in 8 bits: %d entries are outside 1..%d", K, FRB_8BIT_MOST_INNER);
    FRB_CHECK_ARG(copies >= 1, "rows in 8 bits: %d places a row", copies);
    FRB_CHECK_ARG(((uintptr_t)codes & 15) == 0, "rows in 8 bits: codes start on 16 bytes");
    const int KP = up_to(K, FRB_8BIT_KBLOCK);
    // 16-byte loads where every row starts on 16 bytes and its last run of 8 entries ends before the next
    const int whole = x_stride % 8 == 0 && ((uintptr_t)x & 15) == 0;
#define LAUNCH(PER_ROW)                                                                                                          \
    do {                                                                                                                         \
        const int at_once = PER_ROW < 128 ? 128 / PER_ROW : 1, blocks = (rows + at_once - 1) / at_once;                          \
        launch_dependent(rows_8bit_kernel<T, PER_ROW>, dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)),                  \
                         dim3(PER_ROW < 128 ? 128 : PER_ROW), 0, stream, (const T*)x, x_stride, rows, K, KP, places, copies, places ? rows * copies : rows, (int8_t*)codes, scales, whole, (int)early); \
    } while (0)
    // as few threads a row as hold it in registers, where there are rows for every SM and it is no longer than 8,192 entries; else as many as there may be
    FRB_DISPATCH_DTYPE(x_type, T, {
        if (rows <= 2 * frb_sm_count() || K > 256 * 8 * kept_runs(256)) LAUNCH(512);
        else if (K > 128 * 8 * kept_runs(128)) LAUNCH(256);
        else if (K > 64 * 8 * kept_runs(64)) LAUNCH(128);
        else if (K > 32 * 8 * kept_runs(32)) LAUNCH(64);
        else LAUNCH(32);
    });
#undef LAUNCH
    FRB_RETURN_LAUNCH("rows_8bit");
}

// ----------------------------------------------------------------------------- lists of the experts' rows

#define PLAN_THREADS 1024
#define PLAN_KEPT 16                   // ids that a thread keeps in registers between the two passes

// One block counts the assignments of every expert, gives each expert its run of rows and its tiles, and every assignment a row of its
// expert's run.  Which of them comes first there is left to chance: every row's results depend on that row alone.  An id that
// names no expert gets the row -1: nothing is computed for it and nothing added.  Bound by the trips to memory and the counters in shared
// memory: 16,384 ids 7 us with the ids read one after another, 5 with all of a thread's asked for at once.
__global__ void __launch_bounds__(PLAN_THREADS)
plan_kernel(const int* __restrict__ ids, int assignments, int experts, int tile_rows, int* __restrict__ offsets, int* __restrict__ row_of_assign,
            int* __restrict__ tile_expert, int* __restrict__ tile_row0, int* __restrict__ num_tiles) {
    extern __shared__ int next_row[];                       // [experts]: counts, then each expert's next row
    __shared__ int warp_rows[32], warp_tiles[32], rows_before, tiles_before;
    wait_for_previous_kernel();
    let_next_kernel_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int kept[PLAN_KEPT];
#pragma unroll
    for (int i = 0; i < PLAN_KEPT; ++i) {
        const int a = i * PLAN_THREADS + threadIdx.x;
        kept[i] = -1;
        if (i * PLAN_THREADS < assignments && a < assignments) kept[i] = ids[a];
    }
    for (int e = threadIdx.x; e < experts; e += PLAN_THREADS) next_row[e] = 0;
    if (threadIdx.x == 0) { rows_before = 0; tiles_before = 0; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PLAN_KEPT; ++i) {
        if (i * PLAN_THREADS >= assignments) break;
        if ((unsigned)kept[i] < (unsigned)experts) atomicAdd(&next_row[kept[i]], 1);
    }
    for (int a = PLAN_KEPT * PLAN_THREADS + threadIdx.x; a < assignments; a += PLAN_THREADS) {
        const int e = ids[a];
        if ((unsigned)e < (unsigned)experts) atomicAdd(&next_row[e], 1);
    }
    __syncthreads();
    for (int base = 0; base < experts; base += PLAN_THREADS) {
        const int e = base + threadIdx.x;
        const int count = e < experts ? next_row[e] : 0, tiles = (count + tile_rows - 1) / tile_rows;
        int rows_to = count, tiles_to = tiles;              // sums up to and with this expert
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int r = __shfl_up_sync(0xffffffffu, rows_to, o), t = __shfl_up_sync(0xffffffffu, tiles_to, o);
            if (lane >= o) { rows_to += r; tiles_to += t; }
        }
        if (lane == 31) { warp_rows[warp] = rows_to; warp_tiles[warp] = tiles_to; }
        __syncthreads();
        int row = rows_before + rows_to - count, tile = tiles_before + tiles_to - tiles;
        for (int w = 0; w < warp; ++w) { row += warp_rows[w]; tile += warp_tiles[w]; }
        __syncthreads();                                    // all have read the sums before
        if (threadIdx.x == PLAN_THREADS - 1) { rows_before = row + count; tiles_before = tile + tiles; }
        if (e < experts) {
            offsets[e] = row;
            next_row[e] = row;
            for (int i = 0; i < tiles; ++i) { tile_expert[tile + i] = e; tile_row0[tile + i] = row + i * tile_rows; }
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) { offsets[experts] = rows_before; num_tiles[0] = tiles_before; }
#pragma unroll
    for (int i = 0; i < PLAN_KEPT; ++i) {
        const int a = i * PLAN_THREADS + threadIdx.x;
        if (i * PLAN_THREADS >= assignments) break;
        if (a < assignments) row_of_assign[a] = (unsigned)kept[i] < (unsigned)experts ? atomicAdd(&next_row[kept[i]], 1) : -1;
    }
    for (int a = PLAN_KEPT * PLAN_THREADS + threadIdx.x; a < assignments; a += PLAN_THREADS) {
        const int e = ids[a];
        row_of_assign[a] = (unsigned)e < (unsigned)experts ? atomicAdd(&next_row[e], 1) : -1;
    }
}

int plan(const int* ids, int tokens, int top_k, int experts, int tile_rows, int* offsets, int* row_of_assign, int* tile_expert, int* tile_row0,
         int* num_tiles, cudaStream_t stream) {
    launch_dependent(plan_kernel, dim3(1), dim3(PLAN_THREADS), (size_t)experts * sizeof(int), stream, ids, tokens * top_k, experts, tile_rows, offsets,
                     row_of_assign, tile_expert, tile_row0, num_tiles);
    FRB_RETURN_LAUNCH("experts_8bit");
}

// ----------------------------------------------------------------------------- the sum over a token's experts

// out[t] = sum over r of weights[t, r] * y[row_of_assign[t, r]] in the order of r, in float32 and rounded once; a rank without a row adds
// nothing.  Bound by reading y: 16,384 float32 rows of 2048 in 26 us.  (With y in bfloat16 where the results are, 2,048 tokens of 8 experts of 2048
// and 1024 took 174 us instead of 192, and the results were 1.4 times as far from those in 64 bits: not done.)
template <typename OutT, int V>
__global__ void __launch_bounds__(256)
combine_8bit_kernel(const float* __restrict__ y, int y_stride, const float* __restrict__ weights, const int* __restrict__ row_of_assign, int top_k, int width,
                    OutT* __restrict__ out) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    const size_t t = blockIdx.x;
    const int c = (blockIdx.y * 256 + threadIdx.x) * V;
    if (c >= width) return;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
#pragma unroll 4
    for (int r = 0; r < top_k; ++r) {
        const int row = row_of_assign[t * top_k + r];
        if (row < 0) continue;
        const float w = weights[t * top_k + r];
        const float* src = y + (size_t)row * y_stride + c;
        if constexpr (V == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src);
            sum[0] += w * v.x; sum[1] += w * v.y; sum[2] += w * v.z; sum[3] += w * v.w;
        } else {
            sum[0] += w * src[0];
        }
    }
    if constexpr (V == 4) store4(out + t * width + c, make_float4(sum[0], sum[1], sum[2], sum[3]));
    else out[t * width + c] = from_f32<OutT>(sum[0]);
}

int combine(const float* y, int y_stride, const float* weights, const int* row_of_assign, int tokens, int top_k, int width, void* out, int out_type,
            cudaStream_t stream) {
    const bool fours = width % 4 == 0 && y_stride % 4 == 0 && (((uintptr_t)y | (uintptr_t)out) & 15) == 0;
    const dim3 grid((unsigned)tokens, (unsigned)((width + (fours ? 1023 : 255)) / (fours ? 1024 : 256)));
    FRB_CHECK_ARG(grid.y <= 65535, "experts in 8 bits: a width of %d exceeds the grid", width);
    FRB_DISPATCH_DTYPE(out_type, OutT, {
        if (fours) launch_dependent(combine_8bit_kernel<OutT, 4>, grid, dim3(256), 0, stream, y, y_stride, weights, row_of_assign, top_k, width, (OutT*)out);
        else launch_dependent(combine_8bit_kernel<OutT, 1>, grid, dim3(256), 0, stream, y, y_stride, weights, row_of_assign, top_k, width, (OutT*)out);
    });
    FRB_RETURN_LAUNCH("experts_8bit");
}

}  // namespace frb_products8

// Rows of x [rows, K] (float32 or bfloat16) as codes [.., K up to 128] and scales; row t goes to places[t * copies + c], or to row t.
FRB_API int frb_rows_8bit(const void* x, int x_type, int rows, int K, const int* places, int copies, void* codes, float* scales, cudaStream_t stream) {
    return frb_products8::rows_codes(x, x_type, K, rows, K, places, copies, codes, scales, false, stream);
}
