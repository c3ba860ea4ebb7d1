// gnnx_norm.hpp — layer norm (ReLU before it, gain / offset, their gradients), dropout from a counter-based generator, and the two in one
// pass: the run between two graph convolutions of an encoder (models.py:230-267: ReLU, norm; :58-61: the next layer's dropout).
//
// x is a matrix of `rows` rows and `cols` columns, the elements of a row contiguous, the rows x_stride elements apart; v = max(x, 0) or x.
//   forward    mu = mean v, var = mean (v - mu)^2, rstd = (var + eps)^-1/2, xhat = (v - mu) rstd, y = xhat w + b, d = dropout(y)
//   backward   dy = dL/dy + dropout(dL/dd), g = dy w, c1 = mean g, c2 = mean g xhat, dx = rstd (g - c1 - xhat c2) [x > 0],
//              dw = sum over rows of dy xhat, db = sum over rows of dy
//   dropout    word(r, c) = word c mod 4 of Philox-4x32-10 at counter (c / 4, r mod 2^32, r / 2^32, step) under the key `seed`; the element stays,
//              scaled by 1 / (1 - p), where word >= round(p 2^32), and is 0 otherwise.  Recomputed wherever it is needed, never stored.
// All arithmetic in fp32 whatever the storage type (fp32, bf16, fp16); one rounding, at the store.
#pragma once
#include <stdint.h>

namespace gnnx {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

struct DropArgs {
    int32_t on;              // 0: nothing is dropped (threshold 0)
    uint32_t last_dropped;   // threshold - 1: a word is dropped where word <= last_dropped
    float scale;
    uint32_t k0, k1, step;
    const int64_t* state;    // device (seed, step) or null: read when the kernel runs; `step` is added to it
    int64_t row0;            // the row of the whole tensor that row 0 here is
};

struct NormArgs {
    int64_t rows, cols, x_stride, dy_stride, dd_stride;
    const void *x, *w, *b, *dy, *dd;
    void *y, *d, *dx, *dw, *db;
    float *mean, *rstd;
    float eps, relu_floor;   // v = x < relu_floor ? relu_floor : x (0, or -inf without ReLU; NaN stays NaN)
    int32_t relu;
    int32_t w_is_f32;        // type of w, b, dw, db: 1 fp32, 0 the type of x
    float* part;             // [parts][2][cols] partial column sums of the backward pass
    int32_t parts;
    DropArgs drop;
};

struct Philox4 { uint32_t w[4]; };

// Philox-4x32-10: Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011 (the constants are the paper's).
__device__ __forceinline__ Philox4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

struct DropKey { uint32_t k0, k1, step; };
__device__ __forceinline__ DropKey drop_key(const DropArgs& a) {
    if (!a.state) return {a.k0, a.k1, a.step};
    const uint64_t seed = (uint64_t)a.state[0];
    return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)((uint64_t)a.state[1] + a.step)};
}
// the four words of columns 4 block .. 4 block + 3 of row r
__device__ __forceinline__ Philox4 drop_words(const DropArgs& a, const DropKey& k, int64_t r, uint32_t block) {
    const uint64_t row = (uint64_t)(r + a.row0);
    return philox(block, (uint32_t)row, (uint32_t)(row >> 32), k.step, k.k0, k.k1);
}
__device__ __forceinline__ float dropped(const DropArgs& a, uint32_t word, float v) {
    return word > a.last_dropped || !a.on ? v * a.scale : 0.0f;
}

__device__ __forceinline__ float floored(float v, float floor) { return v < floor ? floor : v; }      // ReLU (floor 0) or nothing (floor -inf); NaN stays

template <class T>
__device__ __forceinline__ float param_at(const void* p, int32_t is_f32, int64_t c) {
    return is_f32 ? static_cast<const float*>(p)[c] : (float)static_cast<const T*>(p)[c];
}

// ---- a row in registers ----
// A row is shared by TPR lanes (beyond 64: threads of a workgroup); each holds K pieces of 16 bytes, V elements.  Piece k of lane l is meant to start at column
// (k TPR + l) V; one that would reach past the row starts at cols - V instead and leaves out of every sum the `skip` elements that the piece before it has as
// well (a piece wholly beyond the row leaves out all V).  So every access is one 16-byte access inside the row, whatever the row's length and alignment (the
// hardware takes any alignment): no tail, no variant for odd rows or slices.  Both holders of an element store the same value.  Needs cols >= V.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <class T>
struct Piece {
    static constexpr int V = 16 / (int)sizeof(T);
    u32x4 w;
    __device__ __forceinline__ float at(int j) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, +w[j]);      // (+: of the lane's value; a cast of the vector's lane itself reads lane 0)
        else if constexpr (__is_same(T, bf16_t)) return __builtin_bit_cast(float, j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
        else return (float)__builtin_bit_cast(f16_t, (uint16_t)(j & 1 ? w[j >> 1] >> 16 : w[j >> 1]));
    }
};
template <class T>
__device__ __forceinline__ Piece<T> load_piece(const T* p) {
    Piece<T> q;
    __builtin_memcpy(&q.w, p, 16);
    return q;
}
template <class T>
__device__ __forceinline__ void store_piece(T* p, const float* v) {
    Piece<T> q;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) q.w[j] = __builtin_bit_cast(uint32_t, v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            q.w[j] = (uint32_t)__builtin_bit_cast(uint16_t, (T)v[2 * j]) | (uint32_t)__builtin_bit_cast(uint16_t, (T)v[2 * j + 1]) << 16;
    }
    __builtin_memcpy(p, &q.w, 16);
}
// the V parameters of a piece (fp32, or x's type)
template <class T>
__device__ __forceinline__ void load_params(float* out, const void* p, int32_t is_f32, int64_t c) {
    constexpr int V = Piece<T>::V;
    if (sizeof(T) == 4 || is_f32) {
#pragma unroll
        for (int h = 0; h < V; h += 4) {
            const Piece<float> q = load_piece(static_cast<const float*>(p) + c + h);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[h + j] = q.at(j);
        }
    } else {
        const Piece<T> q = load_piece(static_cast<const T*>(p) + c);
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = q.at(j);
    }
}
struct Slot { int64_t c; int skip; };
template <int V>
__device__ __forceinline__ Slot slot_at(int64_t c, int64_t cols) {
    const int64_t last = cols - V, over = c - last;
    return over <= 0 ? Slot{c, 0} : Slot{last, over < V ? (int)over : V};
}

// The dropout of a piece's V elements from column c on (c is a multiple of 4 unless the piece was moved back from the end of a row that 4 does not divide:
// its words then lie across V / 4 + 1 blocks).
template <class T>
__device__ __forceinline__ void drop_piece(const DropArgs& d, const DropKey& key, int64_t r, int64_t c, int64_t cols, float* v) {
    constexpr int V = Piece<T>::V;
    if ((cols & 3) == 0) {
#pragma unroll
        for (int h = 0; h < V; h += 4) {
            const Philox4 q = drop_words(d, key, r, (uint32_t)(c >> 2) + h / 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[h + j] = dropped(d, q.w[j], v[h + j]);
        }
    } else {
        uint32_t w[V + 4];
#pragma unroll
        for (int h = 0; h < V + 4; h += 4) {
            const Philox4 q = drop_words(d, key, r, (uint32_t)(c >> 2) + h / 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[h + j] = q.w[j];
        }
        const int sh = (int)(c & 3);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t w0 = w[j], w1 = w[j + 1], w2 = w[j + 2], w3 = w[j + 3];      // (values: a choice between the elements would index memory)
            const uint32_t lo = sh & 1 ? w1 : w0, hi = sh & 1 ? w3 : w2;
            v[j] = dropped(d, sh & 2 ? hi : lo, v[j]);
        }
    }
}

// Sums over the TPR lanes that share a row, in every one of them; beyond a wave through `part` (one float per wave and sum).
template <int TPR, int N>
__device__ __forceinline__ void row_totals(float (&v)[N], float (*part)[N]) {
#pragma unroll
    for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) part[threadIdx.x >> 6][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += part[w][i];
            v[i] = s;
        }
    }
}

// y (and d) of one piece from its xhat
template <class T, bool DROP>
__device__ __forceinline__ void norm_outputs(const NormArgs& a, const DropKey& key, int64_t r, int64_t c, float* v) {
    constexpr int V = Piece<T>::V;
    float p[V];
    if (a.w) {
        load_params<T>(p, a.w, a.w_is_f32, c);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= p[j];
    }
    if (a.b) {
        load_params<T>(p, a.b, a.w_is_f32, c);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += p[j];
    }
    if (a.y) store_piece(static_cast<T*>(a.y) + r * a.cols + c, v);
    if (DROP) {
        drop_piece<T>(a.drop, key, r, c, a.cols, v);
        store_piece(static_cast<T*>(a.d) + r * a.cols + c, v);
    }
}

template <int TPR>
constexpr int norm_threads() { return TPR <= 64 ? 256 : TPR; }

template <class T, int TPR, int K, bool DROP>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_norm_forward(NormArgs a) {
    constexpr int V = Piece<T>::V, RPB = norm_threads<TPR>() / TPR;
    __shared__ float part[2][TPR > 64 ? TPR / 64 : 1][1];
    const int l = threadIdx.x % TPR;
    const float inv = 1.0f / (float)a.cols;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const bool live = r0 + threadIdx.x / TPR < a.rows;      // (a workgroup of one row is live as a whole)
        const int64_t r = live ? r0 + threadIdx.x / TPR : a.rows - 1;
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
        Piece<T> q[K];                             // as stored: widened again in each pass, half the registers for 16-bit types
        Slot at[K];
        float s[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            at[k] = slot_at<V>((k * TPR + l) * V, a.cols);
            q[k] = load_piece(x + at[k].c);
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float v = floored(q[k].at(j), a.relu_floor);
                s[0] += 2 * k + 1 < K || j >= at[k].skip ? v : 0.0f;      // (more than half of the K rounds are full: run_forward)
            }
        row_totals<TPR>(s, part[0]);
        const float mean = s[0] * inv;
        s[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float v = floored(q[k].at(j), a.relu_floor) - mean;
                s[0] += 2 * k + 1 < K || j >= at[k].skip ? v * v : 0.0f;
            }
        row_totals<TPR>(s, part[1]);
        const float rstd = 1.0f / sqrtf(s[0] * inv + a.eps);
        if (!live) continue;
        if (l == 0 && a.mean) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (at[k].skip < V) {
                float v[V];
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = (floored(q[k].at(j), a.relu_floor) - mean) * rstd;
                norm_outputs<T, DROP>(a, key, r, at[k].c, v);
            }
        }
    }
}

// Rows too long for registers: one workgroup per row, the row read again for each of the three passes (mean, squared distance from it, output).
template <class T, bool DROP>
__global__ __launch_bounds__(1024) void k_norm_forward_long(NormArgs a) {
    constexpr int V = Piece<T>::V;
    __shared__ float part[2][16][1];
    const float inv = 1.0f / (float)a.cols;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
        float s[1] = {0.0f};
        for (int64_t c = (int64_t)threadIdx.x * V; c < a.cols; c += 1024 * V) {
            const Slot t = slot_at<V>(c, a.cols);
            const Piece<T> q = load_piece(x + t.c);
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += j >= t.skip ? floored(q.at(j), a.relu_floor) : 0.0f;
        }
        row_totals<1024>(s, part[0]);
        const float mean = s[0] * inv;
        s[0] = 0.0f;
        for (int64_t c = (int64_t)threadIdx.x * V; c < a.cols; c += 1024 * V) {
            const Slot t = slot_at<V>(c, a.cols);
            const Piece<T> q = load_piece(x + t.c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float v = floored(q.at(j), a.relu_floor) - mean;
                s[0] += j >= t.skip ? v * v : 0.0f;
            }
        }
        row_totals<1024>(s, part[1]);
        const float rstd = 1.0f / sqrtf(s[0] * inv + a.eps);
        if (threadIdx.x == 0 && a.mean) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        for (int64_t c = (int64_t)threadIdx.x * V; c < a.cols; c += 1024 * V) {
            const Slot t = slot_at<V>(c, a.cols);
            const Piece<T> q = load_piece(x + t.c);
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (floored(q.at(j), a.relu_floor) - mean) * rstd;
            norm_outputs<T, DROP>(a, key, r, t.c, v);
        }
    }
}

// Rows shorter than one piece (fewer than 4 or 8 columns): one thread per row.
template <class T, bool DROP>
__global__ __launch_bounds__(256) void k_norm_forward_narrow(NormArgs a) {
    const float inv = 1.0f / (float)a.cols;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < a.rows; r += (int64_t)gridDim.x * 256) {
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
        float s = 0.0f;
        for (int c = 0; c < a.cols; ++c) s += floored((float)x[c], a.relu_floor);
        const float mean = s * inv;
        s = 0.0f;
        for (int c = 0; c < a.cols; ++c) {
            const float v = floored((float)x[c], a.relu_floor) - mean;
            s += v * v;
        }
        const float rstd = 1.0f / sqrtf(s * inv + a.eps);
        if (a.mean) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        for (int c = 0; c < a.cols; ++c) {
            float v = (floored((float)x[c], a.relu_floor) - mean) * rstd;
            if (a.w) v *= param_at<T>(a.w, a.w_is_f32, c);
            if (a.b) v += param_at<T>(a.b, a.w_is_f32, c);
            if (a.y) static_cast<T*>(a.y)[r * a.cols + c] = (T)v;
            if (DROP) static_cast<T*>(a.d)[r * a.cols + c] = (T)dropped(a.drop, drop_words(a.drop, key, r, (uint32_t)(c >> 2)).w[c & 3], v);
        }
    }
}

__device__ __forceinline__ float wave_total(float v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// dL/dy at (r, c): the gradient of the kept output plus that of the dropped one
template <class T, bool DROP>
__device__ __forceinline__ float norm_dy(const NormArgs& a, const DropKey& key, int64_t r, int64_t c) {
    float g = a.dy ? (float)static_cast<const T*>(a.dy)[r * a.dy_stride + c] : 0.0f;
    if (DROP) g += dropped(a.drop, drop_words(a.drop, key, r, (uint32_t)(c >> 2)).w[c & 3], (float)static_cast<const T*>(a.dd)[r * a.dd_stride + c]);
    return g;
}

template <class T, bool DROP>
__global__ __launch_bounds__(256) void k_norm_backward_rows(NormArgs a) {
    const int lane = threadIdx.x & 63;
    const float inv = 1.0f / (float)a.cols;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.rows; r += (int64_t)gridDim.x * 4) {
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t c = lane; c < a.cols; c += 64) {
            float v = (float)x[c], g = norm_dy<T, DROP>(a, key, r, c);
            v = ((v < a.relu_floor ? a.relu_floor : v) - mean) * rstd;
            if (a.w) g *= param_at<T>(a.w, a.w_is_f32, c);
            s1 += g;
            s2 += g * v;
        }
        const float c1 = wave_total(s1) * inv, c2 = wave_total(s2) * inv;
        for (int64_t c = lane; c < a.cols; c += 64) {
            const float xv = (float)x[c];
            float v = xv, g = norm_dy<T, DROP>(a, key, r, c);
            v = ((v < a.relu_floor ? a.relu_floor : v) - mean) * rstd;
            if (a.w) g *= param_at<T>(a.w, a.w_is_f32, c);
            g = rstd * (g - c1 - v * c2);
            static_cast<T*>(a.dx)[r * a.cols + c] = (T)(a.relu && xv <= 0.0f ? 0.0f : g);
        }
    }
}

// Partial column sums: workgroup (column tile of 64, part) adds the rows r = 4 part + wave mod 4 parts; the four waves join in LDS.
template <class T, bool DROP>
__global__ __launch_bounds__(256) void k_norm_backward_cols(NormArgs a) {
    __shared__ float sums[2][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tiles = (a.cols + 63) / 64;
    const int64_t part = blockIdx.x / tiles, c = (blockIdx.x % tiles) * 64 + lane;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    float sw = 0.0f, sb = 0.0f;
    if (c < a.cols)
        for (int64_t r = part * 4 + wave; r < a.rows; r += (int64_t)a.parts * 4) {
            float v = (float)(static_cast<const T*>(a.x)[r * a.x_stride + c]);
            const float g = norm_dy<T, DROP>(a, key, r, c);
            v = ((v < a.relu_floor ? a.relu_floor : v) - a.mean[r]) * a.rstd[r];
            sw += g * v;
            sb += g;
        }
    sums[0][wave][lane] = sw;
    sums[1][wave][lane] = sb;
    __syncthreads();
    if (wave < 2 && c < a.cols) a.part[(part * 2 + wave) * a.cols + c] = (sums[wave][0][lane] + sums[wave][1][lane]) + (sums[wave][2][lane] + sums[wave][3][lane]);
}

// The backward pass of rows in registers: one pass over x, dy (and dd), dx out.  COLS: a workgroup walks rows a grid apart and keeps its share of dw and db in
// registers; at the end the lanes that hold the same column add up (lane swaps, then LDS across the waves) and the workgroup leaves one partial row of each.
template <class T, int TPR, int K, bool DROP, bool COLS>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_norm_backward(NormArgs a) {
    constexpr int V = Piece<T>::V, RPB = norm_threads<TPR>() / TPR;
    __shared__ float part[2][TPR > 64 ? TPR / 64 : 1][2];
    const int l = threadIdx.x % TPR;
    const float inv = 1.0f / (float)a.cols;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    Slot at[K];
    float sw[K][V], sb[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        at[k] = slot_at<V>((k * TPR + l) * V, a.cols);
#pragma unroll
        for (int j = 0; j < V; ++j) sw[k][j] = sb[k][j] = 0.0f;
    }
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB, turn ^= 1) {
        const bool live = r0 + threadIdx.x / TPR < a.rows;
        const int64_t r = live ? r0 + threadIdx.x / TPR : a.rows - 1;
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
        Piece<T> q[K];
        float g[K][V], s[2] = {0.0f, 0.0f};
        const float mean = a.mean[r], rstd = a.rstd[r];
#pragma unroll
        for (int k = 0; k < K; ++k) q[k] = load_piece(x + at[k].c);
        if (a.dy) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const Piece<T> p = load_piece(static_cast<const T*>(a.dy) + r * a.dy_stride + at[k].c);
#pragma unroll
                for (int j = 0; j < V; ++j) g[k][j] = p.at(j);
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) g[k][j] = 0.0f;
        }
        if (DROP) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const Piece<T> p = load_piece(static_cast<const T*>(a.dd) + r * a.dd_stride + at[k].c);
                float d[V];
#pragma unroll
                for (int j = 0; j < V; ++j) d[j] = p.at(j);
                drop_piece<T>(a.drop, key, r, at[k].c, a.cols, d);
#pragma unroll
                for (int j = 0; j < V; ++j) g[k][j] += d[j];
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float p[V];
            if (a.w) load_params<T>(p, a.w, a.w_is_f32, at[k].c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xhat = (floored(q[k].at(j), a.relu_floor) - mean) * rstd;
                const bool mine = (2 * k + 1 < K || j >= at[k].skip) && (RPB == 1 || live);
                if (COLS) {
                    sb[k][j] += mine ? g[k][j] : 0.0f;
                    sw[k][j] += mine ? g[k][j] * xhat : 0.0f;
                }
                if (a.w) g[k][j] *= p[j];
                s[0] += mine ? g[k][j] : 0.0f;
                s[1] += mine ? g[k][j] * xhat : 0.0f;
            }
        }
        if (!a.dx) continue;
        row_totals<TPR>(s, part[turn]);
        const float c1 = s[0] * inv, c2 = s[1] * inv;
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (at[k].skip < V) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float xv = q[k].at(j), xhat = (floored(xv, a.relu_floor) - mean) * rstd, d = rstd * (g[k][j] - c1 - xhat * c2);
                    g[k][j] = a.relu && xv <= 0.0f ? 0.0f : d;
                }
                store_piece(static_cast<T*>(a.dx) + r * a.cols + at[k].c, g[k]);
            }
        }
    }
    if constexpr (COLS) {
        if constexpr (TPR < 64) {
#pragma unroll
            for (int o = TPR; o < 64; o <<= 1)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    sw[0][j] += __shfl_xor(sw[0][j], o);
                    sb[0][j] += __shfl_xor(sb[0][j], o);
                }
        }
        const int wave = threadIdx.x >> 6;
        __shared__ float lds[RPB > 1 ? 3 : 1][2][RPB > 1 ? V : 1][RPB > 1 ? TPR : 1];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if constexpr (RPB > 1) {
                if (k) __syncthreads();
                if (wave && (threadIdx.x & 63) < TPR)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        lds[wave - 1][0][j][l] = sw[k][j];
                        lds[wave - 1][1][j][l] = sb[k][j];
                    }
                __syncthreads();
                if (threadIdx.x >= TPR) continue;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    sw[k][j] = (sw[k][j] + lds[0][0][j][l]) + (lds[1][0][j][l] + lds[2][0][j][l]);
                    sb[k][j] = (sb[k][j] + lds[0][1][j][l]) + (lds[1][1][j][l] + lds[2][1][j][l]);
                }
            }
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j >= at[k].skip) {
                    a.part[(int64_t)blockIdx.x * 2 * a.cols + at[k].c + j] = sw[k][j];
                    a.part[((int64_t)blockIdx.x * 2 + 1) * a.cols + at[k].c + j] = sb[k][j];
                }
        }
    }
}

// The partial sums of a column: 32 columns and 32 parts at a time per workgroup, each of the 32 sums in part order, then the 32 in order.
template <class T>
__global__ __launch_bounds__(1024) void k_norm_join(NormArgs a) {
    __shared__ float sums[32][33];
    const int64_t i = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31), n = 2 * a.cols;      // dw's columns, then db's
    float s = 0.0f;
    if (i < n) {
#pragma unroll 8
        for (int p = threadIdx.x >> 5; p < a.parts; p += 32) s += a.part[(int64_t)p * n + i];
    }
    sums[threadIdx.x >> 5][threadIdx.x & 31] = s;
    __syncthreads();
    if (threadIdx.x >= 32 || i >= n) return;
    s = 0.0f;
#pragma unroll
    for (int p = 0; p < 32; ++p) s += sums[p][threadIdx.x];
    void* out = i >= a.cols ? a.db : a.dw;
    const int64_t c = i >= a.cols ? i - a.cols : i;
    if (!out) return;
    if (a.w_is_f32) static_cast<float*>(out)[c] = s;
    else static_cast<T*>(out)[c] = (T)s;
}

// One thread per four columns of a row.
template <class T>
__global__ __launch_bounds__(256) void k_dropout(int64_t rows, int64_t cols, int64_t stride, const T* x, T* y, DropArgs d) {
    const DropKey key = drop_key(d);
    const int64_t blocks = (cols + 3) / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * blocks; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / blocks, k = i % blocks;
        Philox4 q = {};
        if (d.on) q = drop_words(d, key, r, (uint32_t)k);
        for (int j = 0; j < 4; ++j) {
            const int64_t c = 4 * k + j;
            if (c >= cols) break;
            const float v = (float)x[r * stride + c];
            y[r * cols + c] = (T)dropped(d, q.w[j], v);
        }
    }
}

}  // namespace gnnx
