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

// No contraction by the compiler: every fma below is written out, so the variants of one launch shape (with or without dropout, with or without the parameters'
// gradients) round an element alike.  (Another launch shape, as rows cut into chunks, takes the row's sums in another order.)
#pragma clang fp contract(off)

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
    float eps;
    float relu_floor;        // v = maximum(x, relu_floor): 0 (then dx = 0 where x <= 0), or -inf without ReLU
    int32_t w_is_f32;        // type of w, b, dw, db: 1 fp32, 0 the type of x
    float* part;             // [parts][2][cols] partial sums of dw and db
    int32_t parts;
    float* chunk;            // long rows: [rows][chunks][2] partial sums of the chunks of a row
    int32_t chunks;
    DropArgs drop;
};

struct Philox4 { uint32_t w[4]; };

// a ^ b ^ c in one instruction
#if defined(__HIPCC__)
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }
#else
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return a ^ b ^ c; }      // (the host compiler of the tests' emulator)
#endif

// Philox-4x32-10: Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011 (the constants are the paper's).
__device__ __forceinline__ Philox4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = xor3((uint32_t)(p1 >> 32), c1, k0);
        c2 = xor3((uint32_t)(p0 >> 32), c3, k1);
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// The value is needed here (no instruction): what it is computed from may not move behind.
#ifndef GNNX_OPAQUE
#define GNNX_OPAQUE(x) asm volatile("" : "+v"(x))
#endif

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
__device__ __forceinline__ bool kept(const DropArgs& a, uint32_t word) { return word > a.last_dropped || !a.on; }
__device__ __forceinline__ float dropped(const DropArgs& a, uint32_t word, float v) { return kept(a, word) ? v * a.scale : 0.0f; }

__device__ __forceinline__ float floored(float v, float floor) { return __builtin_elementwise_maximum(v, floor); }      // ReLU or nothing; NaN stays NaN

// (variance + eps)^-1/2: the hardware's reciprocal square root (within one ulp), its argument kept out of the subnormal numbers it takes for 0
__device__ __forceinline__ float reciprocal_deviation(float v) {
    const bool tiny = v < 0x1p-96f;
    const float y = __builtin_amdgcn_rsqf(tiny ? v * 0x1p96f : v);
    return tiny ? y * 0x1p48f : y;
}

template <class T>
__device__ __forceinline__ float param_at(const void* p, int32_t is_f32, int64_t c) {
    return is_f32 ? static_cast<const float*>(p)[c] : (float)static_cast<const T*>(p)[c];
}

// ---- a row in registers ----
// A row is shared by TPR lanes (beyond 64: threads of a workgroup); each holds K pieces of 16 bytes, V elements.  Piece k of lane l is meant to start at column
// (k TPR + l) V; one that would reach past the row starts at cols - V instead and leaves out of every sum the `skip` elements that the piece before it has as
// well (a piece wholly beyond the row leaves out all V).  So every access is one 16-byte access inside the row, whatever the row's length and alignment (the
// hardware takes any alignment): no tail, no variant for odd rows or slices, no branch around a store - both holders of an element compute and store the same
// bits, and so do lanes whose row lies beyond the last, which repeat that one.  Needs cols >= V.  K is the least that holds the row: only the last round of
// pieces can reach past it.
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
// (column c of a row: a 32-bit byte offset from the row's start, which is the same for a whole wave in all but the narrow shapes - one scalar base per row)
template <class T>
__device__ __forceinline__ Piece<T> load_piece(const void* row, uint32_t c) {
    Piece<T> q;
    __builtin_memcpy(&q.w, static_cast<const char*>(row) + c * (uint32_t)sizeof(T), 16);
    return q;
}
template <class T>
__device__ __forceinline__ void store_piece(void* row, uint32_t c, const float* v) {
    Piece<T> q;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) q.w[j] = __builtin_bit_cast(uint32_t, v[j]);
    } else {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int j = 0; j < 4; ++j) {      // two at a time: one conversion instruction per word
            const f32x2 pair = {v[2 * j], v[2 * j + 1]};
            q.w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, t2));
        }
    }
    __builtin_memcpy(static_cast<char*>(row) + c * (uint32_t)sizeof(T), &q.w, 16);
}
// the V parameters (of type P: fp32, or x's type) of a piece of x
template <class T, class P>
struct Params {
    static constexpr int N = (int)(sizeof(P) / sizeof(T));
    Piece<P> q[N];
    __device__ __forceinline__ void load(const void* p, uint32_t c) {
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = load_piece<P>(p, c + i * Piece<P>::V);
    }
    __device__ __forceinline__ void ones() { fill(sizeof(P) == 4 ? 0x3f800000u : __is_same(P, bf16_t) ? 0x3f803f80u : 0x3c003c00u); }
    __device__ __forceinline__ void zeros() { fill(0u); }
    __device__ __forceinline__ void fill(uint32_t v) {
#pragma unroll
        for (int i = 0; i < N; ++i) q[i].w = (u32x4)v;
    }
    __device__ __forceinline__ float at(int j) const { return q[j / Piece<P>::V].at(j % Piece<P>::V); }
};
struct Slot { uint32_t c; int skip; };
template <int V>
__device__ __forceinline__ Slot slot_at(uint32_t c, uint32_t cols) {      // cols < 2^30
    const int over = (int)c - (int)(cols - V);
    return over <= 0 ? Slot{c, 0} : Slot{cols - V, over < V ? over : V};
}

// The words of a piece's V elements from column c on (c is a multiple of 4 unless the piece was moved back from the end of a row that 4 does not divide: its words
// then lie across V / 4 + 1 blocks).  They need nothing of the data: a kernel forms them while its loads are on their way, and compares them where it needs the
// answer (truth values of more than one piece held that long are packed into bytes by the compiler, at 6 instructions each).  put(j, word): takes the word of element j.
template <class T, class Put>
__device__ __forceinline__ void each_word(const DropArgs& d, const DropKey& key, int64_t r, uint32_t c, uint32_t cols, const Put& put) {
    constexpr int V = Piece<T>::V;
    if ((cols & 3) == 0) {
#pragma unroll
        for (int h = 0; h < V; h += 4) {
            const Philox4 q = drop_words(d, key, r, (c >> 2) + h / 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) put(h + j, q.w[j]);
        }
    } else {
        uint32_t w[V + 4];
#pragma unroll
        for (int h = 0; h < V + 4; h += 4) {
            const Philox4 q = drop_words(d, key, r, (c >> 2) + h / 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[h + j] = q.w[j];
        }
        const int sh = (int)(c & 3);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t w0 = w[j], w1 = w[j + 1], w2 = w[j + 2], w3 = w[j + 3];      // (values: a choice between the elements would index memory)
            const uint32_t lo = sh & 1 ? w1 : w0, hi = sh & 1 ? w3 : w2;
            put(j, sh & 2 ? hi : lo);
        }
    }
}
template <class T>
__device__ __forceinline__ void piece_words(const DropArgs& d, const DropKey& key, int64_t r, uint32_t c, uint32_t cols, uint32_t* out) {
    each_word<T>(d, key, r, c, cols, [out](int j, uint32_t word) { out[j] = word; });
}

// all ones in the bits of a piece's elements that count (all but the first `skip`)
template <class T>
__device__ __forceinline__ u32x4 piece_mask(int skip) {
    u32x4 m;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) m[j] = j >= skip ? ~0u : 0u;
        else m[j] = (2 * j >= skip ? 0xffffu : 0u) | (2 * j + 1 >= skip ? 0xffff0000u : 0u);
    }
    return m;
}

// v + v of lane ^ O (O = 1, 2), of the lane mirrored in its 8 (O = 4) or 16 (O = 8) lanes - the same sum once the smaller groups hold theirs -, of lane ^ O
template <int O>
__device__ __forceinline__ float lane_pair_sum(float v) {
    constexpr int ctrl = O == 1 ? 0xB1 : O == 2 ? 0x4E : O == 4 ? 0x141 : 0x140;
    if constexpr (O > 8) return v + __shfl_xor(v, O);
    else return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, 0xf, 0xf, true));
}
template <int TPR>
__device__ __forceinline__ float lanes_total(float v) {
    if constexpr (TPR > 1) v = lane_pair_sum<1>(v);
    if constexpr (TPR > 2) v = lane_pair_sum<2>(v);
    if constexpr (TPR > 4) v = lane_pair_sum<4>(v);
    if constexpr (TPR > 8) v = lane_pair_sum<8>(v);
    if constexpr (TPR == 32) v = lane_pair_sum<16>(v);
    if constexpr (TPR == 64) {      // the four 16-lane sums through scalar registers: no trip through LDS
        const int i = __builtin_bit_cast(int, v);
        const float q0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 0)), q1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 16));
        const float q2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 32)), q3 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 48));
        v = (q0 + q1) + (q2 + q3);
    }
    return v;
}
// Sums over the TPR lanes that share a row, in every one of them; beyond a wave through `part`, one entry per wave of at most 16 and sum (two calls in a row need
// two), which the 16 lanes of a DPP row read and add at once.  Entries of waves that the workgroup lacks hold 0: clear_part, before the first call.
// WHOLE: however many waves the workgroup has.
constexpr int WHOLE = 1024;
template <int TPR, int M, int N>
__device__ __forceinline__ void clear_part(float (&part)[M][16][N]) {
    if constexpr (TPR > 64) {
        for (int i = threadIdx.x; i < M * 16 * N; i += (int)blockDim.x) (&part[0][0][0])[i] = 0.0f;
        __syncthreads();
    }
}
template <int TPR, int N>
__device__ __forceinline__ void row_totals(float (&v)[N], float (*part)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_total<(TPR < 64 ? TPR : 64)>(v[i]);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) part[threadIdx.x >> 6][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = lanes_total<16>(part[threadIdx.x & 15][i]);
    }
}

// y (and d) of one piece from its xhat; keep(j): whether element j stays
template <class T, class P, bool DROP, class Keep>
__device__ __forceinline__ void norm_outputs(const NormArgs& a, int64_t r, uint32_t c, const Params<T, P>& w, const Params<T, P>& b, const Keep& keep, float* v) {
    constexpr int V = Piece<T>::V;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = __builtin_fmaf(v[j], w.at(j), b.at(j));
    if (a.y) store_piece<T>(static_cast<T*>(a.y) + r * a.cols, c, v);
    if (DROP) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = keep(j) ? v[j] * a.drop.scale : 0.0f;
        store_piece<T>(static_cast<T*>(a.d) + r * a.cols, c, v);
    }
}

// the row of a lane among those its workgroup works on at once
template <int TPR>
__device__ __forceinline__ int row_in_group() {
    if constexpr (TPR > 64) return 0;
    else if constexpr (TPR == 64) return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    else return (int)(threadIdx.x / TPR);
}

// ... and the row itself: the last one for lanes beyond it
template <int TPR>
__device__ __forceinline__ int64_t row_of(int64_t r0, int64_t rows) {
    const int64_t r = r0 + row_in_group<TPR>();
    return r < rows ? r : rows - 1;
}

template <int TPR>
constexpr int norm_threads() { return TPR <= 64 ? 256 : TPR; }

// sum of a lane's K pieces, and of their squared distances from `mean`; FULL: every element of every piece counts (the row is TPR K V long), else those that another
// piece has as well are left out
template <bool FULL, class T, int K>
__device__ __forceinline__ float pieces_sum(const Piece<T> (&q)[K], const Slot (&at)[K], float floor) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        Piece<T> p = q[k];
        if (!FULL && k + 1 == K) p.w &= piece_mask<T>(at[k].skip);
#pragma unroll
        for (int j = 0; j < Piece<T>::V; ++j) s += floored(p.at(j), floor);
    }
    return s;
}
template <bool FULL, class T, int K>
__device__ __forceinline__ float pieces_squares(const Piece<T> (&q)[K], const Slot (&at)[K], float floor, float mean) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < Piece<T>::V; ++j) {
            const float v = floored(q[k].at(j), floor) - mean;
            s = FULL || k + 1 < K || j >= at[k].skip ? __builtin_fmaf(v, v, s) : s;
        }
    return s;
}

// The forward pass: one read of x, mean and then the squared distances from it out of the registers (no E[v^2] - mean^2), one write of each output.
// Bound by HBM: 65536 x 1024 fp32 90 us = 5.96 TB/s, bf16 (fp32 parameters) 46 us = 5.8, 16384 x 4096 bf16 41 us = 6.6 - a copy reaches 6.1.  One row per group of
// lanes and no walk over rows: a grid that covers all rows at once streams better than workgroups that stride (copies: 6.1 against 4.4 to 5.6 TB/s).  With a second,
// dropped output the generator's 40 instructions per four elements fill what the loads leave (65536 x 1024 bf16: 74 us, the VALU busy 69 % of the time, 512 columns
// 39 us and 75 %; fp32 137 us = 5.9 TB/s, 35 %).
template <class T, class P, int TPR, int K, bool DROP>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_norm_forward(NormArgs a) {
    constexpr int V = Piece<T>::V, RPB = norm_threads<TPR>() / TPR;
    __shared__ float part[2][16][1];
    clear_part<TPR>(part);
    const int l = threadIdx.x % TPR;
    const bool full = a.cols == TPR * K * V;
    const float inv = 1.0f / (float)a.cols;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = row_of<TPR>(r0, a.rows);
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
        Piece<T> q[K];                             // as stored: widened again in each pass, half the registers for 16-bit types
        Params<T, P> w[K], b[K];                   // on their way with the row: nothing of the chain load - mean - variance - store waits for them
        Slot at[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            at[k] = slot_at<V>((k * TPR + l) * V, (uint32_t)a.cols);
            q[k] = load_piece<T>(x, at[k].c);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (a.w) w[k].load(a.w, at[k].c);
            else w[k].ones();
            if (a.b) b[k].load(a.b, at[k].c);
            else b[k].zeros();
        }
        uint32_t words[K][V];
        bool flags[V];
        if constexpr (DROP && K == 1) {
            // one piece: lane masks in scalar registers, compared where the words are formed (65536 x 512 bf16 39.4 us, 256 columns 20.7; 41.0 and 21.6 where the
            // words leave the generator's two branches first, 41.2 and 22.0 with words held)
            each_word<T>(a.drop, key, r, at[0].c, (uint32_t)a.cols, [&](int j, uint32_t word) { flags[j] = kept(a.drop, word); });
        } else if constexpr (DROP) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                piece_words<T>(a.drop, key, r, at[k].c, (uint32_t)a.cols, words[k]);
#pragma unroll
                for (int j = 0; j < V; ++j) GNNX_OPAQUE(words[k][j]);      // before the wait for the row: left alone they move behind the reductions
            }
        }
        float s[1];
        if (full) s[0] = pieces_sum<true>(q, at, a.relu_floor);
        else s[0] = pieces_sum<false>(q, at, a.relu_floor);
        row_totals<TPR>(s, part[0]);
        const float mean = s[0] * inv;
        if (full) s[0] = pieces_squares<true>(q, at, a.relu_floor, mean);
        else s[0] = pieces_squares<false>(q, at, a.relu_floor, mean);
        row_totals<TPR>(s, part[1]);
        const float rstd = reciprocal_deviation(s[0] * inv + a.eps);
        if (l == 0 && a.mean) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (floored(q[k].at(j), a.relu_floor) - mean) * rstd;
            norm_outputs<T, P, DROP>(a, r, at[k].c, w[k], b[k], [&](int j) { return K == 1 ? flags[j] : kept(a.drop, words[k][j]); }, v);
        }
    }
}

// ---- rows too long for a workgroup's registers: cut into chunks of CHUNK_LANES x CHUNK_PIECES pieces, a workgroup each, in two launches ----
constexpr int CHUNK_LANES = 256, CHUNK_PIECES = 1;
template <class T>
constexpr int chunk_cols() { return CHUNK_LANES * CHUNK_PIECES * Piece<T>::V; }
// the slots of a lane in chunk `ch`; every chunk but a row's last is full
template <class T>
__device__ __forceinline__ void chunk_slots(Slot (&at)[CHUNK_PIECES], int ch, int64_t cols) {
#pragma unroll
    for (int k = 0; k < CHUNK_PIECES; ++k)
        at[k] = slot_at<Piece<T>::V>((uint32_t)ch * chunk_cols<T>() + (k * CHUNK_LANES + threadIdx.x) * Piece<T>::V, (uint32_t)cols);
}

// x is read twice (forward) and x, dy twice (backward), the second time from the caches where they hold it; a workgroup per row left most of the chip idle and read
// the row three times (48 x 65537 fp32, both passes: 787 us; in chunks 30).  A long row's two statistics are 8 bytes per chunk.
// First launch of the forward pass: the chunk's mean and its sum of squared distances from that mean.
template <class T>
__global__ __launch_bounds__(CHUNK_LANES) void k_norm_chunk_stats(NormArgs a) {
    __shared__ float part[2][16][1];
    clear_part<CHUNK_LANES>(part);
    const int64_t units = a.rows * a.chunks;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t r = u / a.chunks;
        const int ch = (int)(u % a.chunks);
        Slot at[CHUNK_PIECES];
        Piece<T> q[CHUNK_PIECES];
        chunk_slots<T>(at, ch, a.cols);
#pragma unroll
        for (int k = 0; k < CHUNK_PIECES; ++k) q[k] = load_piece<T>(static_cast<const T*>(a.x) + r * a.x_stride, at[k].c);
        float s[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < CHUNK_PIECES; ++k) {
            Piece<T> p = q[k];
            p.w &= piece_mask<T>(at[k].skip);
#pragma unroll
            for (int j = 0; j < Piece<T>::V; ++j) s[0] += floored(p.at(j), a.relu_floor);
        }
        row_totals<CHUNK_LANES>(s, part[0]);
        const int64_t left = a.cols - (int64_t)ch * chunk_cols<T>();
        const float mean = s[0] / (float)(left < chunk_cols<T>() ? left : chunk_cols<T>());
        s[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < CHUNK_PIECES; ++k)
#pragma unroll
            for (int j = 0; j < Piece<T>::V; ++j) {
                const float v = floored(q[k].at(j), a.relu_floor) - mean;
                s[0] = j >= at[k].skip ? __builtin_fmaf(v, v, s[0]) : s[0];
            }
        row_totals<CHUNK_LANES>(s, part[1]);
        if (threadIdx.x == 0) {
            a.chunk[2 * u] = mean;
            a.chunk[2 * u + 1] = s[0];
        }
    }
}

// Second launch: the row's statistics from its chunks' - sum of squares = sum of the chunks' + their sizes times the squared distance of their means from the
// row's - in every workgroup alike, then the chunk's outputs.
template <class T, class P, bool DROP>
__global__ __launch_bounds__(CHUNK_LANES) void k_norm_chunk_outputs(NormArgs a) {
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    const int64_t units = a.rows * a.chunks;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t r = u / a.chunks;
        const int ch = (int)(u % a.chunks);
        Slot at[CHUNK_PIECES];
        Piece<T> q[CHUNK_PIECES];
        chunk_slots<T>(at, ch, a.cols);
#pragma unroll
        for (int k = 0; k < CHUNK_PIECES; ++k) q[k] = load_piece<T>(static_cast<const T*>(a.x) + r * a.x_stride, at[k].c);
        const float* st = a.chunk + 2 * r * a.chunks;
        const int lane = threadIdx.x & 63;
        float s = 0.0f;
        for (int i = lane; i < a.chunks; i += 64) {
            const int64_t left = a.cols - (int64_t)i * chunk_cols<T>();
            s += st[2 * i] * (float)(left < chunk_cols<T>() ? left : chunk_cols<T>());
        }
        const float mean = lanes_total<64>(s) / (float)a.cols;
        s = 0.0f;
        for (int i = lane; i < a.chunks; i += 64) {
            const int64_t left = a.cols - (int64_t)i * chunk_cols<T>();
            const float d = st[2 * i] - mean;
            s += st[2 * i + 1] + d * d * (float)(left < chunk_cols<T>() ? left : chunk_cols<T>());
        }
        const float rstd = reciprocal_deviation(lanes_total<64>(s) / (float)a.cols + a.eps);
        if (ch == 0 && threadIdx.x == 0 && a.mean) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
#pragma unroll
        for (int k = 0; k < CHUNK_PIECES; ++k) {
            float v[Piece<T>::V];
#pragma unroll
            for (int j = 0; j < Piece<T>::V; ++j) v[j] = (floored(q[k].at(j), a.relu_floor) - mean) * rstd;
            Params<T, P> w, b;
            if (a.w) w.load(a.w, at[k].c);
            else w.ones();
            if (a.b) b.load(a.b, at[k].c);
            else b.zeros();
            uint32_t words[Piece<T>::V];
            if (DROP) piece_words<T>(a.drop, key, r, at[k].c, (uint32_t)a.cols, words);
            norm_outputs<T, P, DROP>(a, r, at[k].c, w, b, [&](int j) { return kept(a.drop, words[j]); }, v);
        }
    }
}

// Rows shorter than one piece (fewer than 4 or 8 columns): one thread per row, element by element (10^6 x 7 bf16: 24 us = 1.2 TB/s, bound by the 2-byte accesses).
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
            s = __builtin_fmaf(v, v, s);
        }
        const float rstd = reciprocal_deviation(s * inv + a.eps);
        if (a.mean) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        for (int h = 0; h < a.cols; h += 4) {
            Philox4 q = {};
            if (DROP) q = drop_words(a.drop, key, r, (uint32_t)(h >> 2));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = h + j;
                if (c >= a.cols) break;
                float v = (floored((float)x[c], a.relu_floor) - mean) * rstd;
                const float w = a.w ? param_at<T>(a.w, a.w_is_f32, c) : 1.0f;
                v = a.b ? __builtin_fmaf(v, w, param_at<T>(a.b, a.w_is_f32, c)) : v * w;
                if (a.y) static_cast<T*>(a.y)[r * a.cols + c] = (T)v;
                if (DROP) static_cast<T*>(a.d)[r * a.cols + c] = (T)dropped(a.drop, q.w[j], v);
            }
        }
    }
}

// ---- backward ----
// What a lane holds of one row: its pieces of x, dy and dd as stored.
template <class T, int K, bool DROP>
struct RowPieces {
    static constexpr int V = Piece<T>::V;
    Piece<T> x[K], dy[K], dd[DROP ? K : 1];
    float mean, rstd;
    __device__ __forceinline__ void load(const NormArgs& a, const Slot (&at)[K], int64_t r) {
#pragma unroll
        for (int k = 0; k < K; ++k) x[k] = load_piece<T>(static_cast<const T*>(a.x) + r * a.x_stride, at[k].c);
        if constexpr (DROP) {
#pragma unroll
            for (int k = 0; k < K; ++k) dd[k] = load_piece<T>(static_cast<const T*>(a.dd) + r * a.dd_stride, at[k].c);
        }
        if (!DROP || a.dy) {
#pragma unroll
            for (int k = 0; k < K; ++k) dy[k] = load_piece<T>(static_cast<const T*>(a.dy) + r * a.dy_stride, at[k].c);
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) dy[k].w = (u32x4)0u;
        }
        mean = a.mean[r];
        rstd = a.rstd[r];
    }
    // the dropped output's share of dL/dy, formed once per row
    __device__ __forceinline__ void dropped_share(const NormArgs& a, const DropKey& key, const Slot (&at)[K], int64_t r, float (&d)[DROP ? K : 1][V]) const {
        if constexpr (DROP) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                uint32_t words[V];
                piece_words<T>(a.drop, key, r, at[k].c, (uint32_t)a.cols, words);
#pragma unroll
                for (int j = 0; j < V; ++j) d[k][j] = dropped(a.drop, words[j], dd[k].at(j));
            }
        }
    }
    __device__ __forceinline__ float xhat(const NormArgs& a, int k, int j) const { return (floored(x[k].at(j), a.relu_floor) - mean) * rstd; }
    // dL/dy of piece k: MASKED, 0 in the elements that do not count here
    template <bool MASKED>
    __device__ __forceinline__ void gradient(int k, const u32x4& mask, int skip, const float (&d)[DROP ? K : 1][V], float* g) const {
        Piece<T> p = dy[k];
        if (MASKED) p.w &= mask;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            g[j] = p.at(j);
            if constexpr (DROP) g[j] += !MASKED || j >= skip ? d[k][j] : 0.0f;
        }
    }
    // dx of piece k from the row's rstd c1, rstd c2
    template <class P>
    __device__ __forceinline__ void store_dx(const NormArgs& a, int k, const Slot& at, int64_t r, const Params<T, P>& w, float c1, float c2,
                                             const float (&d)[DROP ? K : 1][V]) const {
        float g[V];
        gradient<false>(k, (u32x4)0u, 0, d, g);
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] = __builtin_fmaf(xhat(a, k, j), -c2, __builtin_fmaf(g[j] * w.at(j), rstd, -c1));
        if (a.relu_floor == 0.0f) {
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] = x[k].at(j) <= 0.0f ? 0.0f : g[j];
        }
        store_piece<T>(static_cast<T*>(a.dx) + r * a.cols, at.c, g);
    }
};

// a lane's partial sums of dw and db, of the columns that count with it
template <int V>
__device__ __forceinline__ void store_cols(const NormArgs& a, int64_t part, const Slot& at, const float* sw, const float* sb) {
    float* out = a.part + part * 2 * a.cols + at.c;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j >= at.skip) {
            out[j] = sw[j];
            out[a.cols + j] = sb[j];
        }
}

// The backward pass of rows in registers: one pass over x, dy (and dd), dx out.  COLS: a workgroup walks rows a grid apart and keeps its share of dw and db in
// registers; at the end the lanes that hold the same column add up (lane sums, then LDS across the waves) and the workgroup leaves one partial row of each.
// Bound by HBM at fp32 (65536 x 1024: 145 us = 5.6 TB/s), at 16 bits by HBM and 164 instructions per piece together (80 us = 5.2 TB/s with the VALU busy 44 % of the
// time; 5 us more are the join of the partial rows).
// The next row is always on its way while one is worked on (the last one is loaded again at the end: a load that may or may not have been issued would make
// the wait for the row before it a wait for everything).
template <class T, class P, int TPR, int K, bool DROP, bool COLS>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_norm_backward(NormArgs a) {
    constexpr int V = Piece<T>::V, RPB = norm_threads<TPR>() / TPR;      // (WHOLE: one row, as many waves as hold it)
    __shared__ float part[2][16][2];
    clear_part<TPR>(part);
    const int l = threadIdx.x % TPR, lanes = TPR == WHOLE ? (int)blockDim.x : TPR;
    const float inv = 1.0f / (float)a.cols;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    Slot at[K];
    Params<T, P> w[K];
    float sw[K][V], sb[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        at[k] = slot_at<V>((k * lanes + l) * V, (uint32_t)a.cols);
        if (a.w) w[k].load(a.w, at[k].c);
        else w[k].ones();
#pragma unroll
        for (int j = 0; j < V; ++j) sw[k][j] = sb[k][j] = 0.0f;
    }
    const u32x4 mask = piece_mask<T>(at[K - 1].skip);
    const int64_t step = (int64_t)gridDim.x * RPB;
    const auto work = [&](const RowPieces<T, K, DROP>& now, int64_t r0, int turn) {
        const int64_t r = row_of<TPR>(r0, a.rows);
        const bool live = r0 + row_in_group<TPR>() < a.rows;
        float d[DROP ? K : 1][V], s[2] = {0.0f, 0.0f};
        now.dropped_share(a, key, at, r, d);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float g[V], xhat[V];
            if (k + 1 < K) now.template gradient<false>(k, mask, 0, d, g);
            else now.template gradient<true>(k, mask, at[k].skip, d, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                xhat[j] = now.xhat(a, k, j);
                const float gw = g[j] * w[k].at(j);
                s[0] += gw;
                s[1] = __builtin_fmaf(gw, xhat[j], s[1]);
            }
            if (COLS && (RPB == 1 || live))
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    sb[k][j] += g[j];
                    sw[k][j] = __builtin_fmaf(g[j], xhat[j], sw[k][j]);
                }
        }
        row_totals<TPR>(s, part[turn]);
        const float c1 = s[0] * inv * now.rstd, c2 = s[1] * inv * now.rstd;
#pragma unroll
        for (int k = 0; k < K; ++k) now.store_dx(a, k, at[k], r, w[k], c1, c2, d);
    };
    RowPieces<T, K, DROP> even, odd;
    int64_t r0 = (int64_t)blockIdx.x * RPB;
    if (r0 < a.rows) {
        even.load(a, at, row_of<TPR>(r0, a.rows));
        for (;;) {
            odd.load(a, at, row_of<TPR>(r0 + step, a.rows));
            work(even, r0, 0);
            if ((r0 += step) >= a.rows) break;
            even.load(a, at, row_of<TPR>(r0 + step, a.rows));
            work(odd, r0, 1);
            if ((r0 += step) >= a.rows) break;
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
            store_cols<V>(a, blockIdx.x, at[k], sw[k], sb[k]);
        }
    }
}

// Long rows, first launch of the backward pass: a chunk's sums of g and g xhat.
template <class T, class P, bool DROP>
__global__ __launch_bounds__(CHUNK_LANES) void k_norm_chunk_sums(NormArgs a) {
    constexpr int V = Piece<T>::V, K = CHUNK_PIECES;
    __shared__ float part[2][16][2];
    clear_part<CHUNK_LANES>(part);
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    const int64_t units = a.rows * a.chunks;
    int turn = 0;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x, turn ^= 1) {
        const int64_t r = u / a.chunks;
        Slot at[K];
        chunk_slots<T>(at, (int)(u % a.chunks), a.cols);
        RowPieces<T, K, DROP> now;
        now.load(a, at, r);
        float d[DROP ? K : 1][V], s[2] = {0.0f, 0.0f};
        now.dropped_share(a, key, at, r, d);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float g[V];
            Params<T, P> w;
            if (a.w) w.load(a.w, at[k].c);
            else w.ones();
            now.template gradient<true>(k, piece_mask<T>(at[k].skip), at[k].skip, d, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float gw = g[j] * w.at(j);
                s[0] += gw;
                s[1] = __builtin_fmaf(gw, now.xhat(a, k, j), s[1]);
            }
        }
        row_totals<CHUNK_LANES>(s, part[turn]);
        if (threadIdx.x < 2) a.chunk[2 * u + threadIdx.x] = s[threadIdx.x];
    }
}

// Second launch: workgroup (chunk, part) walks the rows part, part + parts, ...: dx of its chunk, and its share of dw and db.
template <class T, class P, bool DROP, bool COLS>
__global__ __launch_bounds__(CHUNK_LANES) void k_norm_chunk_backward(NormArgs a) {
    constexpr int V = Piece<T>::V, K = CHUNK_PIECES;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    const int ch = (int)(blockIdx.x % (unsigned)a.chunks), lane = threadIdx.x & 63;
    const int64_t first = blockIdx.x / (unsigned)a.chunks, step = gridDim.x / (unsigned)a.chunks;
    const float inv = 1.0f / (float)a.cols;
    Slot at[K];
    chunk_slots<T>(at, ch, a.cols);
    float sw[K][V], sb[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) sw[k][j] = sb[k][j] = 0.0f;
    Params<T, P> w[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (a.w) w[k].load(a.w, at[k].c);
        else w[k].ones();
    }
    // the row's sums are on their way with its pieces, two chunks a lane; more chunks (rows of more than 128) when the row is worked on
    struct Sums { float g[2], x[2]; };
    const auto sums_of = [&](int64_t r) {
        Sums q;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = lane + 64 * h < a.chunks ? lane + 64 * h : a.chunks - 1;
            q.g[h] = a.chunk[2 * (r * a.chunks + i)];
            q.x[h] = a.chunk[2 * (r * a.chunks + i) + 1];
        }
        return q;
    };
    const auto work = [&](const RowPieces<T, K, DROP>& now, const Sums& q, int64_t r) {
        float c1 = lane < a.chunks ? q.g[0] : 0.0f, c2 = lane < a.chunks ? q.x[0] : 0.0f, d[DROP ? K : 1][V];
        if (lane + 64 < a.chunks) {
            c1 += q.g[1];
            c2 += q.x[1];
        }
        for (int i = lane + 128; i < a.chunks; i += 64) {
            c1 += a.chunk[2 * (r * a.chunks + i)];
            c2 += a.chunk[2 * (r * a.chunks + i) + 1];
        }
        now.dropped_share(a, key, at, r, d);
        if (COLS)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float g[V];
                now.template gradient<true>(k, piece_mask<T>(at[k].skip), at[k].skip, d, g);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    sb[k][j] += g[j];
                    sw[k][j] = __builtin_fmaf(g[j], now.xhat(a, k, j), sw[k][j]);
                }
            }
        c1 = lanes_total<64>(c1) * inv * now.rstd;
        c2 = lanes_total<64>(c2) * inv * now.rstd;
#pragma unroll
        for (int k = 0; k < K; ++k) now.store_dx(a, k, at[k], r, w[k], c1, c2, d);
    };
    RowPieces<T, K, DROP> even, odd;
    Sums even_sums, odd_sums;
    int64_t r = first;
    if (r < a.rows) {
        even.load(a, at, r);
        even_sums = sums_of(r);
        for (;;) {
            odd.load(a, at, r + step < a.rows ? r + step : r);
            odd_sums = sums_of(r + step < a.rows ? r + step : r);
            work(even, even_sums, r);
            if ((r += step) >= a.rows) break;
            even.load(a, at, r + step < a.rows ? r + step : r);
            even_sums = sums_of(r + step < a.rows ? r + step : r);
            work(odd, odd_sums, r);
            if ((r += step) >= a.rows) break;
        }
    }
    if constexpr (COLS) {
#pragma unroll
        for (int k = 0; k < K; ++k) store_cols<V>(a, first, at[k], sw[k], sb[k]);
    }
}

// Rows shorter than one piece: one thread per row, its share of dw and db in registers (at most 7 columns), joined over the workgroup in LDS.
template <class T, bool DROP>
__global__ __launch_bounds__(256) void k_norm_backward_narrow(NormArgs a) {
    constexpr int V = Piece<T>::V;
    __shared__ float sums[4][2][V];
    const float inv = 1.0f / (float)a.cols;
    const DropKey key = DROP ? drop_key(a.drop) : DropKey{};
    float sw[V], sb[V];
#pragma unroll
    for (int c = 0; c < V; ++c) sw[c] = sb[c] = 0.0f;
    for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < a.rows; r += (int64_t)gridDim.x * 256) {
        const float mean = a.mean[r], rstd = a.rstd[r];
        float x[V], g[V], c1 = 0.0f, c2 = 0.0f;
#pragma unroll
        for (int c = 0; c < V; ++c) {
            x[c] = g[c] = 0.0f;
            if (c >= a.cols) continue;
            x[c] = (float)static_cast<const T*>(a.x)[r * a.x_stride + c];
            if (a.dy) g[c] = (float)static_cast<const T*>(a.dy)[r * a.dy_stride + c];
            if (DROP)
                g[c] += dropped(a.drop, drop_words(a.drop, key, r, (uint32_t)(c >> 2)).w[c & 3], (float)static_cast<const T*>(a.dd)[r * a.dd_stride + c]);
            const float xhat = (floored(x[c], a.relu_floor) - mean) * rstd;
            sb[c] += g[c];
            sw[c] = __builtin_fmaf(g[c], xhat, sw[c]);
            if (a.w) g[c] *= param_at<T>(a.w, a.w_is_f32, c);
            c1 += g[c];
            c2 = __builtin_fmaf(g[c], xhat, c2);
        }
        c1 *= inv * rstd;
        c2 *= inv * rstd;
#pragma unroll
        for (int c = 0; c < V; ++c)
            if (c < a.cols) {
                const float d = __builtin_fmaf((floored(x[c], a.relu_floor) - mean) * rstd, -c2, __builtin_fmaf(g[c], rstd, -c1));
                static_cast<T*>(a.dx)[r * a.cols + c] = (T)(a.relu_floor == 0.0f && x[c] <= 0.0f ? 0.0f : d);
            }
    }
    if (!a.parts) return;
#pragma unroll
    for (int c = 0; c < V; ++c) {
        sw[c] = lanes_total<64>(sw[c]);
        sb[c] = lanes_total<64>(sb[c]);
        if ((threadIdx.x & 63) == 0) {
            sums[threadIdx.x >> 6][0][c] = sw[c];
            sums[threadIdx.x >> 6][1][c] = sb[c];
        }
    }
    __syncthreads();
    if (threadIdx.x < 2 * V) {
        const int b = threadIdx.x / V, c = threadIdx.x % V;
        if (c < a.cols) a.part[((int64_t)blockIdx.x * 2 + b) * a.cols + c] = (sums[0][b][c] + sums[1][b][c]) + (sums[2][b][c] + sums[3][b][c]);
    }
}

// The partial sums of a column in part order.  MANY: 32 columns and 32 parts at a time per workgroup (each of the 32 sums in part order, then the 32 in four groups), else
// a thread per column - rows so long that they left few partial rows: 7 of 65537 columns 10 us with MANY, 3 without.
template <class T, bool MANY>
__global__ __launch_bounds__(MANY ? 1024 : 256) void k_norm_join(NormArgs a) {
    const int64_t n = 2 * a.cols;      // dw's columns, then db's
    int64_t i;
    float s = 0.0f;
    if constexpr (MANY) {
        __shared__ float sums[32][33];
        i = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
        if (i < n) {
#pragma unroll 8
            for (int p = threadIdx.x >> 5; p < a.parts; p += 32) s += a.part[(int64_t)p * n + i];
        }
        sums[threadIdx.x >> 5][threadIdx.x & 31] = s;
        __syncthreads();
        if (threadIdx.x >= 32) return;
        float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < 32; ++p) q[p & 3] += sums[p][threadIdx.x];
        s = (q[0] + q[1]) + (q[2] + q[3]);
        if (i >= n) return;
    } else {
        i = (int64_t)blockIdx.x * 256 + threadIdx.x;
        if (i >= n) return;
#pragma unroll 8
        for (int p = 0; p < a.parts; ++p) s += a.part[(int64_t)p * n + i];
    }
    void* out = i >= a.cols ? a.db : a.dw;
    const int64_t c = i >= a.cols ? i - a.cols : i;
    if (!out) return;
    if (a.w_is_f32) static_cast<float*>(out)[c] = s;
    else static_cast<T*>(out)[c] = (T)s;
}

// ---- dropout alone ----
struct DropoutArgs {
    int64_t rows, cols, stride;
    const void* x;
    void* y;
    uint32_t pieces, magic, shift;      // pieces of a row; n / pieces = (mulhi(n, magic) + n) >> shift for n < 2^32 (the sum in 33 bits)
    DropArgs drop;
};

// One thread per piece of a row, the words formed before the load returns.  Bound by HBM: 16384 x 4096 bf16 42 us = 6.4 TB/s, 65536 x 1024 fp32 87 us = 6.2 (a copy:
// 6.1); at 16 bits the generator's 10 instructions per element are close behind (the VALU is busy 69 % of the time, 41 % at fp32).  32 bits per element and 10 rounds cost nothing over
// 16 bits or 7 rounds there.  BIG: more pieces in all than 32 bits count.
template <class T, bool BIG>
__global__ __launch_bounds__(256) void k_dropout(DropoutArgs a) {
    constexpr int V = Piece<T>::V;
    const DropKey key = drop_key(a.drop);
    const int64_t n = a.rows * a.pieces;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        int64_t r;
        if (BIG) r = i / a.pieces;
        else r = (uint32_t)((((uint64_t)(uint32_t)i * a.magic >> 32) + (uint32_t)i) >> a.shift);
        const Slot at = slot_at<V>((uint32_t)(i - r * a.pieces) * V, (uint32_t)a.cols);
        const Piece<T> q = load_piece<T>(static_cast<const T*>(a.x) + r * a.stride, at.c);
        float v[V];
        uint32_t words[V];
        piece_words<T>(a.drop, key, r, at.c, (uint32_t)a.cols, words);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = dropped(a.drop, words[j], q.at(j));
        store_piece<T>(static_cast<T*>(a.y) + r * a.cols, at.c, v);
    }
}

// Rows shorter than one piece: one thread per row.
template <class T>
__global__ __launch_bounds__(256) void k_dropout_narrow(DropoutArgs a) {
    const DropKey key = drop_key(a.drop);
    for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < a.rows; r += (int64_t)gridDim.x * 256)
        for (int c = 0; c < a.cols; c += 4) {
            const Philox4 q = drop_words(a.drop, key, r, (uint32_t)(c >> 2));
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < a.cols)
                    static_cast<T*>(a.y)[r * a.cols + c + j] = (T)dropped(a.drop, q.w[j], (float)static_cast<const T*>(a.x)[r * a.stride + c + j]);
        }
}

}  // namespace gnnx
