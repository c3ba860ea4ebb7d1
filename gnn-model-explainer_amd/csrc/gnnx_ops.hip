// gnnx_ops.hip — C ABI (include/gnnx.h) over the encoder-layer operators of gnnx_norm.hpp: layer norm, dropout, and both in one pass.
// Host side only: argument checks, launch shapes.  The library keeps nothing between calls; workspaces are the caller's.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <limits>

#include "../../include/gnnx.h"
#include "gnnx_error.hpp"
#include "gnnx_norm.hpp"

using namespace gnnx;

namespace {

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    char text[256];
    snprintf(text, sizeof(text), "%s: %s", what, hipGetErrorString(e));
    return set_error(text);
}

// workgroups of a launch that walks `items` with a grid stride: at most 2^31 threads in all (the work-items of a launch are counted in 32 bits)
unsigned grid_of(int64_t items, int64_t per_group, int64_t threads) {
    const int64_t g = (items + per_group - 1) / per_group, most = (int64_t(1) << 31) / threads;
    return (unsigned)(g < 1 ? 1 : g > most ? most : g);
}

const char* drop_args(const gnnx_drop* d, DropArgs* out) {
    *out = DropArgs{};
    if (!d) return nullptr;
    if (!(d->p >= 0.0 && d->p <= 1.0)) return "dropout: p must be in [0, 1]";
    const double thr = std::nearbyint(d->p * 4294967296.0);       // 0 .. 2^32, ties to even (Python's round)
    out->on = thr > 0.0;
    out->last_dropped = out->on ? (uint32_t)(thr - 1.0) : 0u;
    out->scale = d->p < 1.0 ? (float)(1.0 / (1.0 - d->p)) : 0.0f;
    out->k0 = (uint32_t)d->seed;
    out->k1 = (uint32_t)(d->seed >> 32);
    out->step = d->step;
    out->state = d->state;
    out->row0 = d->row_offset;
    return nullptr;
}

const char* norm_args(const gnnx_norm* n, NormArgs* a) {
    if (!n) return "null argument";
    if (n->type < 0 || n->type > 2) return "layer norm: type must be 0 (fp32), 1 (bf16) or 2 (fp16)";
    if (n->rows < 0 || n->cols < 1 || n->cols >= (int64_t(1) << 30)) return "layer norm: needs rows >= 0 and 1 <= cols < 2^30";
    if (n->x_stride < 0 || n->dy_stride < 0 || n->dd_stride < 0) return "layer norm: row strides must not be negative";
    if (!(n->eps >= 0.0f)) return "layer norm: eps must not be negative";
    *a = NormArgs{};
    a->rows = n->rows;
    a->cols = n->cols;
    a->x_stride = n->x_stride;
    a->dy_stride = n->dy_stride;
    a->dd_stride = n->dd_stride;
    a->x = n->x;
    a->w = n->w;
    a->b = n->b;
    a->dy = n->dy;
    a->dd = n->dd;
    a->y = n->y;
    a->d = n->d;
    a->dx = n->dx;
    a->dw = n->dw;
    a->db = n->db;
    a->mean = n->mean;
    a->rstd = n->rstd;
    a->eps = n->eps;
    a->relu = n->relu != 0;
    a->relu_floor = n->relu ? 0.0f : -std::numeric_limits<float>::infinity();
    a->w_is_f32 = n->w_is_f32 != 0 || n->type == GNNX_F32;
    return nullptr;
}

// How the backward pass of a row is shared out: lanes per row and pieces per lane; lanes == 0: the row does not fit registers (or is shorter than a piece).
struct RowShape { int lanes, pieces; };
RowShape backward_shape(int32_t type, int64_t cols) {
    const int64_t v = type == GNNX_F32 ? 4 : 8, pieces = (cols + v - 1) / v;
    if (cols < v || pieces > 2048) return {0, 0};
    for (int lanes = 1; lanes <= 64; lanes *= 2)
        if (pieces <= lanes) return {lanes, 1};
    return pieces <= 128 ? RowShape{64, 2} : pieces <= 256 ? RowShape{64, 4} : pieces <= 512 ? RowShape{256, 2} : pieces <= 1024 ? RowShape{256, 4} : RowShape{512, 4};
}

// Partial rows of dw and db: one per workgroup of k_norm_backward, or per slice of the rows of k_norm_backward_cols.
int col_parts(int32_t type, int64_t rows, int64_t cols) {
    const RowShape sh = backward_shape(type, cols);
    int64_t parts;
    if (sh.lanes) {
        const int64_t per = sh.lanes <= 64 ? 256 / sh.lanes : 1, groups = (rows + per - 1) / per;
        parts = groups / 2;
        if (parts > 1024) parts = 1024;
    } else {
        const int64_t tiles = (cols + 63) / 64;
        parts = 2048 / tiles;
        if (parts > (rows + 15) / 16) parts = (rows + 15) / 16;
    }
    return (int)(parts < 1 ? 1 : parts);
}

template <class T, int TPR, int K, bool DROP>
void forward_rows(const NormArgs& a, hipStream_t s) {
    constexpr int NT = norm_threads<TPR>();
    hipLaunchKernelGGL((k_norm_forward<T, TPR, K, DROP>), dim3(grid_of(a.rows, NT / TPR, NT)), dim3(NT), 0, s, a);
}

// The lanes of a row: as few as hold it with one piece each up to a wave, then two to eight pieces each before more waves join in.
template <class T, bool DROP>
void run_forward(const NormArgs& a, hipStream_t s) {
    const int64_t pieces = (a.cols + Piece<T>::V - 1) / Piece<T>::V;
    if (a.cols < Piece<T>::V) hipLaunchKernelGGL((k_norm_forward_narrow<T, DROP>), dim3(grid_of(a.rows, 256, 256)), dim3(256), 0, s, a);
    else if (pieces <= 1) forward_rows<T, 1, 1, DROP>(a, s);
    else if (pieces <= 2) forward_rows<T, 2, 1, DROP>(a, s);
    else if (pieces <= 4) forward_rows<T, 4, 1, DROP>(a, s);
    else if (pieces <= 8) forward_rows<T, 8, 1, DROP>(a, s);
    else if (pieces <= 16) forward_rows<T, 16, 1, DROP>(a, s);
    else if (pieces <= 32) forward_rows<T, 32, 1, DROP>(a, s);
    else if (pieces <= 64) forward_rows<T, 64, 1, DROP>(a, s);
    else if (pieces <= 128) forward_rows<T, 64, 2, DROP>(a, s);
    else if (pieces <= 256) forward_rows<T, 64, 4, DROP>(a, s);
    else if (pieces <= 512) forward_rows<T, 256, 2, DROP>(a, s);
    else if (pieces <= 1024) forward_rows<T, 256, 4, DROP>(a, s);
    else if (pieces <= 2048) forward_rows<T, 1024, 2, DROP>(a, s);
    else if (pieces <= 4096) forward_rows<T, 1024, 4, DROP>(a, s);
    else hipLaunchKernelGGL((k_norm_forward_long<T, DROP>), dim3(grid_of(a.rows, 1, 1024)), dim3(1024), 0, s, a);
}

template <class T, int TPR, int K, bool DROP>
void backward_rows(const NormArgs& a, hipStream_t s) {
    constexpr int NT = norm_threads<TPR>();
    if (a.parts) hipLaunchKernelGGL((k_norm_backward<T, TPR, K, DROP, true>), dim3((unsigned)a.parts), dim3(NT), 0, s, a);
    else if (a.rows) hipLaunchKernelGGL((k_norm_backward<T, TPR, K, DROP, false>), dim3(grid_of(a.rows, NT / TPR, NT)), dim3(NT), 0, s, a);
}

template <class T, bool DROP>
void run_backward(const NormArgs& a, RowShape sh, hipStream_t s) {
    switch (sh.lanes * 8 + sh.pieces) {
        case 1 * 8 + 1: backward_rows<T, 1, 1, DROP>(a, s); break;
        case 2 * 8 + 1: backward_rows<T, 2, 1, DROP>(a, s); break;
        case 4 * 8 + 1: backward_rows<T, 4, 1, DROP>(a, s); break;
        case 8 * 8 + 1: backward_rows<T, 8, 1, DROP>(a, s); break;
        case 16 * 8 + 1: backward_rows<T, 16, 1, DROP>(a, s); break;
        case 32 * 8 + 1: backward_rows<T, 32, 1, DROP>(a, s); break;
        case 64 * 8 + 1: backward_rows<T, 64, 1, DROP>(a, s); break;
        case 64 * 8 + 2: backward_rows<T, 64, 2, DROP>(a, s); break;
        case 64 * 8 + 4: backward_rows<T, 64, 4, DROP>(a, s); break;
        case 256 * 8 + 2: backward_rows<T, 256, 2, DROP>(a, s); break;
        case 256 * 8 + 4: backward_rows<T, 256, 4, DROP>(a, s); break;
        case 512 * 8 + 4: backward_rows<T, 512, 4, DROP>(a, s); break;
        default:
            if (a.dx && a.rows) hipLaunchKernelGGL((k_norm_backward_rows<T, DROP>), dim3(grid_of(a.rows, 4, 256)), dim3(256), 0, s, a);
            if (a.parts) hipLaunchKernelGGL((k_norm_backward_cols<T, DROP>), dim3((unsigned)((a.cols + 63) / 64) * (unsigned)a.parts), dim3(256), 0, s, a);
    }
    if (a.parts) hipLaunchKernelGGL((k_norm_join<T>), dim3((unsigned)((2 * a.cols + 31) / 32)), dim3(1024), 0, s, a);
}

}  // namespace

extern "C" int gnnx_layer_norm_forward(const gnnx_norm* n, const gnnx_drop* drop, void* stream) {
    NormArgs a;
    if (const char* e = norm_args(n, &a)) return set_error(e);
    if (const char* e = drop_args(drop, &a.drop)) return set_error(e);
    if (a.rows == 0) return 0;
    if (!a.y && !a.d) return set_error("layer norm: no output");
    if ((a.d != nullptr) != (drop != nullptr)) return set_error("layer norm: a dropped output and its dropout go together");
    if ((a.mean != nullptr) != (a.rstd != nullptr)) return set_error("layer norm: mean and rstd go together");
    if (!a.x) return set_error("null argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (n->type == GNNX_F32) a.d ? run_forward<float, true>(a, s) : run_forward<float, false>(a, s);
    else if (n->type == GNNX_BF16) a.d ? run_forward<bf16_t, true>(a, s) : run_forward<bf16_t, false>(a, s);
    else a.d ? run_forward<f16_t, true>(a, s) : run_forward<f16_t, false>(a, s);
    return launched("gnnx_layer_norm_forward");
}

extern "C" size_t gnnx_layer_norm_workspace_bytes(int32_t type, int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 1) return 0;
    return (size_t)col_parts(type, rows, cols) * 2 * (size_t)cols * sizeof(float);
}

extern "C" int gnnx_layer_norm_backward(const gnnx_norm* n, const gnnx_drop* drop, void* workspace, size_t workspace_bytes, void* stream) {
    NormArgs a;
    if (const char* e = norm_args(n, &a)) return set_error(e);
    if (const char* e = drop_args(drop, &a.drop)) return set_error(e);
    if (!a.dx && !a.dw && !a.db) return 0;
    if (a.rows > 0 && (a.dd != nullptr) != (drop != nullptr)) return set_error("layer norm: the gradient of a dropped output and its dropout go together");
    if (a.rows > 0 && ((!a.dy && !a.dd) || !a.x || !a.mean || !a.rstd)) return set_error("null argument");
    if (a.dw || a.db) {
        if (!workspace || workspace_bytes < gnnx_layer_norm_workspace_bytes(n->type, a.rows, a.cols)) return set_error("workspace too small");
        a.part = static_cast<float*>(workspace);
        a.parts = col_parts(n->type, a.rows, a.cols);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    const RowShape sh = backward_shape(n->type, a.cols);
    if (n->type == GNNX_F32) a.dd ? run_backward<float, true>(a, sh, s) : run_backward<float, false>(a, sh, s);
    else if (n->type == GNNX_BF16) a.dd ? run_backward<bf16_t, true>(a, sh, s) : run_backward<bf16_t, false>(a, sh, s);
    else a.dd ? run_backward<f16_t, true>(a, sh, s) : run_backward<f16_t, false>(a, sh, s);
    return launched("gnnx_layer_norm_backward");
}

extern "C" int gnnx_dropout(int32_t type, int64_t rows, int64_t cols, const void* x, int64_t x_stride, void* y, const gnnx_drop* drop, void* stream) {
    DropArgs d;
    if (type < 0 || type > 2) return set_error("dropout: type must be 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (!drop) return set_error("null argument");
    if (const char* e = drop_args(drop, &d)) return set_error(e);
    if (rows < 0 || cols < 0 || x_stride < 0 || cols >= (int64_t(1) << 34)) return set_error("dropout: needs rows, stride >= 0 and 0 <= cols < 2^34");
    if (rows == 0 || cols == 0) return 0;
    if (!x || !y) return set_error("null argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid(grid_of(rows * ((cols + 3) / 4), 256, 256)), block(256);
    if (type == GNNX_F32) hipLaunchKernelGGL((k_dropout<float>), grid, block, 0, s, rows, cols, x_stride, static_cast<const float*>(x), static_cast<float*>(y), d);
    else if (type == GNNX_BF16) hipLaunchKernelGGL((k_dropout<bf16_t>), grid, block, 0, s, rows, cols, x_stride, static_cast<const bf16_t*>(x), static_cast<bf16_t*>(y), d);
    else hipLaunchKernelGGL((k_dropout<f16_t>), grid, block, 0, s, rows, cols, x_stride, static_cast<const f16_t*>(x), static_cast<f16_t*>(y), d);
    return launched("gnnx_dropout");
}
