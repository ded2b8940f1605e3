// Products of few rows with 4-bit weights (q4.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ge {

// A Q4_0 or Q4_1 matrix in device memory, in tiles of 16 rows by 128 columns (four groups of 32), rows
// and columns padded with zero weights. Tile t of row block b at index b * (cols_pad / 128) + t:
//   q: 64 lanes x 4 dwords. Lane l's dword g holds row l % 16, columns 32 g + 8 (l / 16) + [0, 8) of the
//     tile: its B operand of one v_mfma_f32_16x16x32. Column 2 i at nibble i, 2 i + 1 at nibble 4 + i.
//   d (and m of Q4_1, w = d q + m; Q4_0 has w = d (q - 8)): fp16 [16 rows][4 groups].
struct Q4Dev {
    int rows = 0, cols = 0, tiles = 0;  // tiles: column tiles of a row block
    uint32_t* q = nullptr;
    uint16_t* d = nullptr;
    uint16_t* m = nullptr;
};

inline int q4_row_blocks(int rows) { return (rows + 15) / 16; }
inline int q4_tiles(int cols) { return (cols + 127) / 128; }

// GGUF blocks in device memory (18 bytes of Q4_0, 20 of Q4_1 where w.m is set) into w's planes.
hipError_t launch_q4_repack(hipStream_t s, const unsigned char* blocks, const Q4Dev& w);

struct Q4Args {
    Q4Dev w, up;        // up: the second matrix of the GeGLU form
    const uint16_t* x;  // [rows][w.cols]
    void* y;            // [rows][w.rows]
    int rows;
};
// Rows of x a call takes (16 or more a workgroup, in the grid's second dimension), and a matrix's rows and
// columns (a workgroup a row block, in the first; columns are counted past the end in 32 bits).
constexpr int kQ4MaxRows = 1 << 19, kQ4MaxWeightRows = 1 << 26, kQ4MaxCols = 1 << 24;
enum Q4Out { kQ4F32 = 0, kQ4F16 = 1, kQ4BF16 = 2 };

// y[r][n] = sum_k x[r][k] w[n][k], or gelu_tanh(x w^T) * (x up^T) with geglu; x fp16 or (bf16) bfloat16.
hipError_t launch_gemv_q4(hipStream_t s, const Q4Args& a, bool bf16, bool geglu, Q4Out out);

}  // namespace ge
