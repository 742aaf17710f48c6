// The rows of a step as warps read them, 32 at a time: which rows a lane looks at.  Plain arithmetic without CUDA, so that the host can go
// through all of it.
#pragma once

#ifdef __CUDACC__
#define FRB_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define FRB_HOST_DEVICE inline
#endif

// Rows in up to `most` groups, each `steps` times 32 rows; the last group's last steps may lie behind the last row.
struct RowGroups { int steps, count; };

FRB_HOST_DEVICE RowGroups row_groups(int rows, int most) {
    const int steps = (rows + 32 * most - 1) / (32 * most);
    return {steps, (rows + 32 * steps - 1) / (32 * steps)};
}

// The row beside the 32 rows from b0 on that a lane looks at besides its own: lane 0 the one in front of them, lane 31 the one behind; -1: none.
FRB_HOST_DEVICE int row_beside(int b0, int lane, int rows) {
    if (b0 >= rows) return -1;
    if (lane == 0) return b0 - 1;
    return lane == 31 && b0 + 32 < rows ? b0 + 32 : -1;
}
