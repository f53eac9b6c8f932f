// Launchers of the ragged products: grouped.hip (by expert), lora.hip (by adapter).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace glmmoe {

struct GroupedArgs {
    const uint16_t* x;        // rows of K values, ldx apart
    long ldx;
    int x_rows;
    const int* row_ids;       // [rows] row of x, or null: row r
    const uint16_t *w0, *w1;  // [E] x [N, K], w_stride apart; w1: the up matrices, or null
    long w_stride;
    const int* off;           // [E + 1]
    const uint16_t *s0, *s1;  // sh_rows > 0: the matrices of group E (the shared expert)
    int sh_row, sh_rows;      // and its rows, after the others'
    int E, rows, N, K;        // rows: those off counts
    void* y;                  // a row for each, ldy apart
    long ldy;
    int ntn;                  // set by the launch: workgroups along N, large tiles in fours
    bool fours;
};
// dtype: kBf16 or kF16 (x and W); f32: y is fp32, else of that type.
int launch_grouped(const GroupedArgs& a, int dtype, bool f32, hipStream_t s);

// Slot-order combine of fp32 rows (topk <= 8, H % 4 == 0).
int launch_grouped_combine(const float* part, const int* inv, const int* ids, const float* w, int n,
                           int topk, int E, int H, int shared, float* out, hipStream_t s);

struct LoraArgs {
    const void* x;            // [n, K], ldx apart
    long ldx;
    const int* ids;           // [n] adapter of each token; outside [0, L): none
    const uint16_t *A, *B;    // [L, r, K], [L, N, r]
    const int* ranks;         // [L] or null: r
    const float* scale;       // [L] or null: 1
    int n, L, K, r, N;
    const void* base;         // [n, N], ldb apart
    long ldb;
    void* y;                  // [n, N], ldy apart
    long ldy;
    float* part;              // lora_part_bytes: [splits][n][rp], A x of each K split
    int splits, kstep, rp;    // set by the launch: K per split, row length of part,
    int jm, je, nx;           // workgroups per token block (by adapter), at both ends; along N
};
size_t lora_part_bytes(int n, int K, int r);
int launch_lora(const LoraArgs& a, int xdt, int wdt, int ydt, hipStream_t s);

}  // namespace glmmoe
