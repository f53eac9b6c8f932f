// C-ABI of the ragged products on 16-bit weights: argument checks and launches.
// Declarations and contracts: include/glmmoe.h.
#include <hip/hip_runtime.h>

#include "../../include/glmmoe.h"
#include "grouped.hpp"

using namespace glmmoe;

namespace {

inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline bool half(int dt) { return dt == GLMMOE_BF16 || dt == GLMMOE_F16; }
inline int64_t size_of(int dt) { return dt == GLMMOE_F32 ? 4 : 2; }

// Whether two [rows, cols] arrays share a byte.
bool overlap(const void* a, int64_t ra, int64_t lda, int64_t ca, int64_t sa, const void* b,
             int64_t rb, int64_t ldb, int64_t cb, int64_t sb) {
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
    const uintptr_t a1 = a0 + ((ra - 1) * lda + ca) * sa, b1 = b0 + ((rb - 1) * ldb + cb) * sb;
    return a0 < b1 && b0 < a1;
}

int grouped(int dtype, const void* x, int64_t ldx, int64_t x_rows, const int* row_ids,
            const void* w0, const void* w1, bool dual, int64_t w_stride, const int* off, int E,
            int64_t rows, int64_t N, int64_t K, int ydt, void* y, int64_t ldy, void* stream) {
    if (!half(dtype) || (ydt != GLMMOE_F32 && ydt != dtype)) return GLMMOE_ERR_ARG;
    if (E <= 0 || rows < 0 || x_rows < 0 || N <= 0 || K <= 0) return GLMMOE_ERR_ARG;
    if (rows == 0) return GLMMOE_OK;
    if (!x || !w0 || (dual && !w1) || !off || !y || x_rows == 0) return GLMMOE_ERR_ARG;
    constexpr int64_t kDim = 1 << 24, kRows = 1 << 30;
    if (E > 4096 || rows >= kRows || x_rows >= kRows || N >= kDim || K >= kDim) return GLMMOE_ERR_SHAPE;
    if (ldx < K || ldy < N || ldx >= kRows || ldy >= kRows || w_stride < 0 ||
        (E > 1 && w_stride < N * K))
        return GLMMOE_ERR_SHAPE;
    if (!row_ids && x_rows < rows) return GLMMOE_ERR_SHAPE;
    if (reinterpret_cast<uintptr_t>(x) % 2 || reinterpret_cast<uintptr_t>(w0) % 2 ||
        reinterpret_cast<uintptr_t>(w1) % 2 || reinterpret_cast<uintptr_t>(y) % size_of(ydt))
        return GLMMOE_ERR_ARG;
    if (overlap(x, x_rows, ldx, K, 2, y, rows, ldy, N, size_of(ydt))) return GLMMOE_ERR_ARG;
    GroupedArgs a{};
    a.x = static_cast<const uint16_t*>(x);
    a.ldx = ldx;
    a.x_rows = (int)x_rows;
    a.row_ids = row_ids;
    a.w0 = static_cast<const uint16_t*>(w0);
    a.w1 = static_cast<const uint16_t*>(w1);
    a.w_stride = w_stride;
    a.off = off;
    a.E = E, a.rows = (int)rows, a.N = (int)N, a.K = (int)K;
    a.y = y;
    a.ldy = ldy;
    return launch_grouped(a, dtype, ydt == GLMMOE_F32, S(stream));
}

bool lora_shape_ok(int n, int L, int64_t K, int r) {
    return n < (1 << 24) && K < (1 << 24) && r <= 256 && L <= (1 << 24);
}

}  // namespace

extern "C" {

int glmmoe_grouped_linear(int dtype, const void* x, int64_t ldx, int64_t x_rows,
                          const int* row_ids, const void* w, int64_t w_stride,
                          const int* expert_offsets, int E, int64_t rows, int64_t N, int64_t K,
                          int y_dtype, void* y, int64_t ldy, void* stream) {
    return grouped(dtype, x, ldx, x_rows, row_ids, w, nullptr, false, w_stride, expert_offsets, E,
                   rows, N, K, y_dtype, y, ldy, stream);
}

int glmmoe_grouped_gate_up(int dtype, const void* x, int64_t ldx, int64_t x_rows,
                           const int* row_ids, const void* w_gate, const void* w_up,
                           int64_t w_stride, const int* expert_offsets, int E, int64_t rows,
                           int64_t N, int64_t K, int h_dtype, void* h, int64_t ldh, void* stream) {
    return grouped(dtype, x, ldx, x_rows, row_ids, w_gate, w_up, true, w_stride, expert_offsets, E,
                   rows, N, K, h_dtype, h, ldh, stream);
}

size_t glmmoe_lora_workspace_bytes(int n, int n_adapters, int64_t K, int r) {
    if (n <= 0 || n_adapters <= 0 || K <= 0 || r <= 0 || !lora_shape_ok(n, n_adapters, K, r)) return 0;
    return lora_part_bytes(n, (int)K, r);
}

int glmmoe_lora_add(int x_dtype, const void* x, int64_t ldx, const int* adapter_ids, int n,
                    int w_dtype, const void* A, const void* B, const int* ranks,
                    const float* scale, int n_adapters, int r, int64_t K, int64_t N, int y_dtype,
                    const void* base, int64_t ldb, void* y, int64_t ldy, void* workspace,
                    size_t workspace_bytes, void* stream) {
    if (!half(w_dtype) || (x_dtype != GLMMOE_F32 && x_dtype != w_dtype) ||
        (y_dtype != GLMMOE_F32 && y_dtype != w_dtype))
        return GLMMOE_ERR_ARG;
    if (n < 0 || n_adapters <= 0 || r <= 0 || K <= 0 || N <= 0) return GLMMOE_ERR_ARG;
    if (n == 0) return GLMMOE_OK;
    if (!x || !adapter_ids || !A || !B || !base || !y) return GLMMOE_ERR_ARG;
    if (!lora_shape_ok(n, n_adapters, K, r) || N >= (1 << 24)) return GLMMOE_ERR_SHAPE;
    constexpr int64_t kLd = 1 << 30;
    if (ldx < K || ldb < N || ldy < N || ldx >= kLd || ldb >= kLd || ldy >= kLd) return GLMMOE_ERR_SHAPE;
    auto off = [](const void* p, int64_t v) { return reinterpret_cast<uintptr_t>(p) % v != 0; };
    const int64_t ys = size_of(y_dtype);
    if (off(x, size_of(x_dtype)) || off(A, 2) || off(B, 2) || off(base, ys) || off(y, ys))
        return GLMMOE_ERR_ARG;
    if ((y != base || ldy != ldb) && overlap(base, n, ldb, N, ys, y, n, ldy, N, ys)) return GLMMOE_ERR_ARG;
    if (!workspace || off(workspace, 16) ||
        workspace_bytes < glmmoe_lora_workspace_bytes(n, n_adapters, K, r))
        return GLMMOE_ERR_WORKSPACE;
    LoraArgs a{};
    a.x = x;
    a.ldx = ldx;
    a.ids = adapter_ids;
    a.A = static_cast<const uint16_t*>(A);
    a.B = static_cast<const uint16_t*>(B);
    a.ranks = ranks;
    a.scale = scale;
    a.n = n, a.L = n_adapters, a.K = (int)K, a.r = r, a.N = (int)N;
    a.base = base;
    a.ldb = ldb;
    a.y = y;
    a.ldy = ldy;
    a.part = static_cast<float*>(workspace);
    return launch_lora(a, x_dtype, w_dtype, y_dtype, S(stream));
}

}  // extern "C"
