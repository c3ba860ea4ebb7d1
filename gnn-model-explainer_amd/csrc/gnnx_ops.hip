// gnnx_ops.hip — C ABI (include/gnnx.h) over the encoder-layer operators of gnnx_norm.hpp: layer norm, dropout, and both in one pass.
// Host side only: argument checks, launch shapes.  The library keeps nothing between calls; workspaces are the caller's.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
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

// Whether an output (contiguous rows) shares memory with a matrix whose rows are `stride` elements apart.  It must not: two lanes may hold one element (a row's last
// piece is moved back into the row, lanes beyond the last row repeat it) and one may read it after the other has stored it.
bool overlap(const void* out, const void* in, int64_t stride, int64_t rows, int64_t cols, int32_t type) {
    if (!out || !in || rows <= 0 || cols <= 0) return false;
    const __int128 size = type == GNNX_F32 ? 4 : 2, row = cols * size, step = stride * size, lo = (__int128)(uintptr_t)out - (__int128)(uintptr_t)in, hi = lo + rows * row;
    if (step == 0) return lo < row && hi > 0;
    const __int128 r = lo < row ? 0 : (lo - row) / step + 1;      // the first row of `in` that ends behind the start of `out`
    return r < rows && r * step < hi && r * step + row > lo;
}
const char* const OVERLAP = "an output shares memory with an input or with the other output";

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
    a->relu_floor = n->relu ? 0.0f : -std::numeric_limits<float>::infinity();
    a->w_is_f32 = n->w_is_f32 != 0 || n->type == GNNX_F32;
    return nullptr;
}

// How a row is shared out: NARROW, shorter than a piece; LONG, cut into chunks; else `lanes` lanes with `pieces` pieces each.
enum { NARROW = 0, LONG = -1 };
struct RowShape { int lanes, pieces; };
int64_t pieces_of(int32_t type, int64_t cols) { return type == GNNX_F32 ? (cols + 3) / 4 : (cols + 7) / 8; }
// As few lanes as hold the row with one piece each up to a wave, then two to four pieces each before more waves join in.
RowShape forward_shape(int32_t type, int64_t cols) {
    const int64_t pieces = pieces_of(type, cols);
    if (cols < (type == GNNX_F32 ? 4 : 8)) return {NARROW, 0};
    for (int lanes = 1; lanes <= 64; lanes *= 2)
        if (pieces <= lanes) return {lanes, 1};
    for (int lanes : {64, 256})
        if (pieces <= 4 * lanes) return {lanes, (int)((pieces + lanes - 1) / lanes)};
    return pieces <= 2048 ? RowShape{1024, 2} : RowShape{LONG, 0};
}
// One piece per lane; rows of more than a wave's pieces take a workgroup of as many waves as hold them.  (Two to four pieces per lane of fewer waves cost registers
// for the sums of dw and db - 8 to 16 per piece and as many again - and were 2 to 20 % slower at 1024 to 8192 columns.)
RowShape backward_shape(int32_t type, int64_t cols) {
    const int64_t pieces = pieces_of(type, cols);
    if (cols < (type == GNNX_F32 ? 4 : 8)) return {NARROW, 0};
    for (int lanes = 1; lanes <= 64; lanes *= 2)
        if (pieces <= lanes) return {lanes, 1};
    if (pieces <= WHOLE) return {(int)((pieces + 63) / 64) * 64, 1};
    return type == GNNX_F32 && pieces <= 2 * WHOLE ? RowShape{(int)((pieces + 127) / 128) * 64, 2} : RowShape{LONG, 0};
}
int chunks_of(int32_t type, int64_t cols) {
    const int64_t per = type == GNNX_F32 ? chunk_cols<float>() : chunk_cols<bf16_t>();
    return (int)((cols + per - 1) / per);
}

// Partial rows of dw and db: one per workgroup that walks rows.
int col_parts(int32_t type, int64_t rows, int64_t cols) {
    const RowShape sh = backward_shape(type, cols);
    int64_t parts;
    if (sh.lanes == LONG) {
        parts = 512 / chunks_of(type, cols);      // two workgroups per CU; 1024: 48 x 65537 fp32 21.1 us for 20.4, 4096 x 16384 bf16 136 for 138
        if (parts > rows / 2) parts = rows / 2;
    } else {
        // Eight waves per CU, in whole workgroups per CU (2.67 of three waves each left a third of the CUs with more to do than the rest: 20011 x 1280 bf16 44 us, 4: 39):
        // more waves gain nothing with a row always in flight, and each workgroup leaves a partial row to write and read again (8192 x 8192 bf16: 256 workgroups
        // 87 us, 512: 103, 1024: 124; 99997 x 20 fp32: 128 15.6 us, 256 11.1, 512 10.1).
        const int64_t threads = sh.lanes <= 64 ? 256 : sh.lanes, per = sh.lanes == NARROW ? 256 : sh.lanes <= 64 ? 256 / sh.lanes : 1, groups = (rows + per - 1) / per;
        const int64_t most = 256 * ((512 + threads - 1) / threads);
        parts = groups / 2;
        if (parts > most) parts = most;
    }
    return (int)(parts < 1 ? 1 : parts);
}

size_t chunk_bytes(int32_t type, int64_t rows, int64_t cols) { return (size_t)rows * (size_t)chunks_of(type, cols) * 2 * sizeof(float); }

size_t workspace_bytes_of(int32_t type, int64_t rows, int64_t cols, bool backward) {
    size_t b = 0;
    if ((backward ? backward_shape(type, cols) : forward_shape(type, cols)).lanes == LONG) b += chunk_bytes(type, rows, cols);
    if (backward) b += (size_t)col_parts(type, rows, cols) * 2 * (size_t)cols * sizeof(float);
    return b;
}

template <class T, class P, int TPR, int K, bool DROP>
void forward_rows(const NormArgs& a, hipStream_t s) {
    constexpr int NT = norm_threads<TPR>();
    hipLaunchKernelGGL((k_norm_forward<T, P, TPR, K, DROP>), dim3(grid_of(a.rows, NT / TPR, NT)), dim3(NT), 0, s, a);
}

template <class T, class P, bool DROP>
void run_forward(const NormArgs& a, RowShape sh, hipStream_t s) {
    const unsigned units = grid_of(a.rows * a.chunks, 1, CHUNK_LANES);
    switch (sh.lanes * 8 + sh.pieces) {
        case 1 * 8 + 1: forward_rows<T, P, 1, 1, DROP>(a, s); break;
        case 2 * 8 + 1: forward_rows<T, P, 2, 1, DROP>(a, s); break;
        case 4 * 8 + 1: forward_rows<T, P, 4, 1, DROP>(a, s); break;
        case 8 * 8 + 1: forward_rows<T, P, 8, 1, DROP>(a, s); break;
        case 16 * 8 + 1: forward_rows<T, P, 16, 1, DROP>(a, s); break;
        case 32 * 8 + 1: forward_rows<T, P, 32, 1, DROP>(a, s); break;
        case 64 * 8 + 1: forward_rows<T, P, 64, 1, DROP>(a, s); break;
        case 64 * 8 + 2: forward_rows<T, P, 64, 2, DROP>(a, s); break;
        case 64 * 8 + 3: forward_rows<T, P, 64, 3, DROP>(a, s); break;
        case 64 * 8 + 4: forward_rows<T, P, 64, 4, DROP>(a, s); break;
        case 256 * 8 + 2: forward_rows<T, P, 256, 2, DROP>(a, s); break;
        case 256 * 8 + 3: forward_rows<T, P, 256, 3, DROP>(a, s); break;
        case 256 * 8 + 4: forward_rows<T, P, 256, 4, DROP>(a, s); break;
        case 1024 * 8 + 2: forward_rows<T, P, 1024, 2, DROP>(a, s); break;
        case NARROW: hipLaunchKernelGGL((k_norm_forward_narrow<T, DROP>), dim3(grid_of(a.rows, 256, 256)), dim3(256), 0, s, a); break;
        default:
            hipLaunchKernelGGL((k_norm_chunk_stats<T>), dim3(units), dim3(CHUNK_LANES), 0, s, a);
            hipLaunchKernelGGL((k_norm_chunk_outputs<T, P, DROP>), dim3(units), dim3(CHUNK_LANES), 0, s, a);
    }
}

template <class T>
constexpr int type_code() { return sizeof(T) == 4 ? GNNX_F32 : GNNX_BF16; }      // (fp16 and bf16 have one geometry)

// (without dw and db the walk over the rows is the same: the next row's load needs rows to come)
template <class T, class P, int TPR, bool DROP, int K = 1>
void backward_rows(const NormArgs& a, int lanes, hipStream_t s) {
    const int threads = TPR == WHOLE ? lanes : 256;
    if (a.parts) hipLaunchKernelGGL((k_norm_backward<T, P, TPR, K, DROP, true>), dim3((unsigned)a.parts), dim3(threads), 0, s, a);
    else if (a.rows) hipLaunchKernelGGL((k_norm_backward<T, P, TPR, K, DROP, false>), dim3((unsigned)col_parts(type_code<T>(), a.rows, a.cols)), dim3(threads), 0, s, a);
}

template <class T, class P, bool DROP>
void run_backward(const NormArgs& a, RowShape sh, hipStream_t s) {
    switch (sh.lanes) {
        case 1: backward_rows<T, P, 1, DROP>(a, 1, s); break;
        case 2: backward_rows<T, P, 2, DROP>(a, 2, s); break;
        case 4: backward_rows<T, P, 4, DROP>(a, 4, s); break;
        case 8: backward_rows<T, P, 8, DROP>(a, 8, s); break;
        case 16: backward_rows<T, P, 16, DROP>(a, 16, s); break;
        case 32: backward_rows<T, P, 32, DROP>(a, 32, s); break;
        case 64: backward_rows<T, P, 64, DROP>(a, 64, s); break;
        case NARROW: hipLaunchKernelGGL((k_norm_backward_narrow<T, DROP>), dim3(a.parts ? (unsigned)a.parts : grid_of(a.rows, 256, 256)), dim3(256), 0, s, a); break;
        default:
            if constexpr (sizeof(T) == 4) {
                if (sh.pieces == 2) {
                    backward_rows<T, P, WHOLE, DROP, 2>(a, sh.lanes, s);
                    break;
                }
            }
            backward_rows<T, P, WHOLE, DROP>(a, sh.lanes, s);
            break;
        case LONG: {
            const unsigned parts = (unsigned)col_parts(type_code<T>(), a.rows, a.cols), grid = (unsigned)a.chunks * parts;
            if (a.rows) hipLaunchKernelGGL((k_norm_chunk_sums<T, P, DROP>), dim3(grid_of(a.rows * a.chunks, 1, CHUNK_LANES)), dim3(CHUNK_LANES), 0, s, a);
            if (a.parts) hipLaunchKernelGGL((k_norm_chunk_backward<T, P, DROP, true>), dim3(grid), dim3(CHUNK_LANES), 0, s, a);
            else if (a.rows) hipLaunchKernelGGL((k_norm_chunk_backward<T, P, DROP, false>), dim3(grid), dim3(CHUNK_LANES), 0, s, a);
        }
    }
    if (a.parts > 16) hipLaunchKernelGGL((k_norm_join<T, true>), dim3((unsigned)((2 * a.cols + 31) / 32)), dim3(1024), 0, s, a);
    else if (a.parts) hipLaunchKernelGGL((k_norm_join<T, false>), dim3((unsigned)((2 * a.cols + 255) / 256)), dim3(256), 0, s, a);
}

template <class T, class P>
void forward(const NormArgs& a, RowShape sh, hipStream_t s) { a.d ? run_forward<T, P, true>(a, sh, s) : run_forward<T, P, false>(a, sh, s); }
template <class T, class P>
void backward(const NormArgs& a, RowShape sh, hipStream_t s) { a.dd ? run_backward<T, P, true>(a, sh, s) : run_backward<T, P, false>(a, sh, s); }

}  // namespace

extern "C" size_t gnnx_layer_norm_workspace_bytes(int32_t type, int64_t rows, int64_t cols, int32_t backward) {
    return type < 0 || type > 2 || rows < 0 || cols < 1 ? 0 : workspace_bytes_of(type, rows, cols, backward != 0);
}

extern "C" int gnnx_layer_norm_forward(const gnnx_norm* n, const gnnx_drop* drop, void* workspace, size_t workspace_bytes, void* stream) {
    NormArgs a;
    if (const char* e = norm_args(n, &a)) return set_error(e);
    if (const char* e = drop_args(drop, &a.drop)) return set_error(e);
    if (a.rows == 0) return 0;
    if (!a.y && !a.d) return set_error("layer norm: no output");
    if ((a.d != nullptr) != (drop != nullptr)) return set_error("layer norm: a dropped output and its dropout go together");
    if ((a.mean != nullptr) != (a.rstd != nullptr)) return set_error("layer norm: mean and rstd go together");
    if (!a.x) return set_error("null argument");
    for (const void* out : {a.y, a.d})
        if (overlap(out, a.x, a.x_stride, a.rows, a.cols, n->type)) return set_error(OVERLAP);
    if (overlap(a.y, a.d, a.cols, a.rows, a.cols, n->type)) return set_error(OVERLAP);
    const RowShape sh = forward_shape(n->type, a.cols);
    if (sh.lanes == LONG) {
        if (!workspace || workspace_bytes < workspace_bytes_of(n->type, a.rows, a.cols, false)) return set_error("workspace too small");
        a.chunk = static_cast<float*>(workspace);
        a.chunks = chunks_of(n->type, a.cols);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (n->type == GNNX_F32) forward<float, float>(a, sh, s);
    else if (n->type == GNNX_BF16) a.w_is_f32 ? forward<bf16_t, float>(a, sh, s) : forward<bf16_t, bf16_t>(a, sh, s);
    else a.w_is_f32 ? forward<f16_t, float>(a, sh, s) : forward<f16_t, f16_t>(a, sh, s);
    return launched("gnnx_layer_norm_forward");
}

extern "C" int gnnx_layer_norm_backward(const gnnx_norm* n, const gnnx_drop* drop, void* workspace, size_t workspace_bytes, void* stream) {
    NormArgs a;
    if (const char* e = norm_args(n, &a)) return set_error(e);
    if (const char* e = drop_args(drop, &a.drop)) return set_error(e);
    if (a.rows > 0 && (a.dd != nullptr) != (drop != nullptr)) return set_error("layer norm: the gradient of a dropped output and its dropout go together");
    if (a.rows > 0 && ((!a.dy && !a.dd) || !a.x || !a.mean || !a.rstd || !a.dx)) return set_error("null argument");
    if (overlap(a.dx, a.x, a.x_stride, a.rows, a.cols, n->type) || overlap(a.dx, a.dy, a.dy_stride, a.rows, a.cols, n->type) ||
        overlap(a.dx, a.dd, a.dd_stride, a.rows, a.cols, n->type))
        return set_error(OVERLAP);
    const RowShape sh = backward_shape(n->type, a.cols);
    const size_t needed = workspace_bytes_of(n->type, a.rows, a.cols, true);
    if ((a.dw || a.db || sh.lanes == LONG) && (!workspace || workspace_bytes < needed)) return set_error("workspace too small");
    if (a.dw || a.db) {
        a.part = static_cast<float*>(workspace);
        a.parts = col_parts(n->type, a.rows, a.cols);
    }
    if (sh.lanes == LONG) {
        a.chunk = reinterpret_cast<float*>(static_cast<char*>(workspace) + (needed - chunk_bytes(n->type, a.rows, a.cols)));
        a.chunks = chunks_of(n->type, a.cols);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (n->type == GNNX_F32) backward<float, float>(a, sh, s);
    else if (n->type == GNNX_BF16) a.w_is_f32 ? backward<bf16_t, float>(a, sh, s) : backward<bf16_t, bf16_t>(a, sh, s);
    else a.w_is_f32 ? backward<f16_t, float>(a, sh, s) : backward<f16_t, f16_t>(a, sh, s);
    return launched("gnnx_layer_norm_backward");
}

namespace {
template <class T>
void run_dropout(const DropoutArgs& a, hipStream_t s) {
    const int64_t n = a.rows * (int64_t)a.pieces;
    if (a.cols < Piece<T>::V) hipLaunchKernelGGL((k_dropout_narrow<T>), dim3(grid_of(a.rows, 256, 256)), dim3(256), 0, s, a);
    else if (n >= (int64_t(1) << 32)) hipLaunchKernelGGL((k_dropout<T, true>), dim3(grid_of(n, 256, 256)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_dropout<T, false>), dim3(grid_of(n, 256, 256)), dim3(256), 0, s, a);
}
}  // namespace

extern "C" int gnnx_dropout(int32_t type, int64_t rows, int64_t cols, const void* x, int64_t x_stride, void* y, const gnnx_drop* drop, void* stream) {
    DropoutArgs a{};
    if (type < 0 || type > 2) return set_error("dropout: type must be 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (!drop) return set_error("null argument");
    if (const char* e = drop_args(drop, &a.drop)) return set_error(e);
    if (rows < 0 || cols < 0 || x_stride < 0 || cols >= (int64_t(1) << 30)) return set_error("dropout: needs rows, stride >= 0 and 0 <= cols < 2^30");
    if (rows == 0 || cols == 0) return 0;
    if (!x || !y) return set_error("null argument");
    if (overlap(y, x, x_stride, rows, cols, type)) return set_error(OVERLAP);
    a.rows = rows;
    a.cols = cols;
    a.stride = x_stride;
    a.x = x;
    a.y = y;
    const uint64_t d = (uint64_t)pieces_of(type, cols);      // < 2^32
    a.pieces = (uint32_t)d;
    // division by d of any n < 2^32: with 2^shift the power of two at or above d, magic = floor(2^32 (2^shift - d) / d) + 1
    while ((uint64_t(1) << a.shift) < d) ++a.shift;
    a.magic = (uint32_t)((((uint64_t(1) << a.shift) - d) << 32) / d + 1);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == GNNX_F32) run_dropout<float>(a, s);
    else if (type == GNNX_BF16) run_dropout<bf16_t>(a, s);
    else run_dropout<f16_t>(a, s);
    return launched("gnnx_dropout");
}
