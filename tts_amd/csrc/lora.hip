// Low-rank adapters of many requests beside a shared projection:
//   y_t = act(base_t + s_k B_k (A_k x_t)),  k = index of the token's segment, and the gradients of it.
//
// With 2 rank operations for every value that is read or written, all of it is bound by memory as long as the factors stay in
// cache and h = A_k x never leaves the workgroup: one launch reads x once, keeps h in registers and adds B_k h to base.
// Products run on the matrix units with tokens as columns (16 x 16 tiles, D[row = 4 (lane / 16) + i][column = lane % 16]), so
// the h that the first product leaves in a lane is the operand that the second one takes from it.
#include "operators.h"

#include <algorithm>

namespace {
using op::ReduceTable;
using op::RunTable;
using op::SegTable;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2_any __attribute__((ext_vector_type(2), aligned(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t raw2 __attribute__((ext_vector_type(2)));
typedef raw2 raw2_any __attribute__((aligned(2)));

// One product step over 16 bytes of k a lane: 32 k of bf16 in one instruction, 16 k of f32 in four.  The k a lane group
// holds are 8 (4) consecutive ones of the operands; both operands agree, which is all that the sum needs.
template <class T> __device__ __forceinline__ f4 product(raw4 a, raw4 b, f4 c);
template <> __device__ __forceinline__ f4 product<bf16_t>(raw4 a, raw4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f4 product<float>(raw4 a, raw4 b, f4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
}
// h as the second product's operand.  f32: itself.  bf16: the 8 places of a lane hold the four values in two parts, and B's
// four values come twice: h = hi + lo to 2^-16 at the price of one instruction (rounded to one part alone, h would cost
// half of the result's own precision).
template <class T> __device__ __forceinline__ raw4 second(f4 h);
template <> __device__ __forceinline__ raw4 second<float>(f4 h) { return __builtin_bit_cast(raw4, h); }
template <> __device__ __forceinline__ raw4 second<bf16_t>(f4 h) {
    raw4 r;
    r[0] = bf16_pair(h[0], h[1]);
    r[1] = bf16_pair(h[2], h[3]);
    r[2] = bf16_pair(h[0] - __uint_as_float(r[0] << 16), h[1] - __uint_as_float(r[0] & 0xffff0000u));
    r[3] = bf16_pair(h[2] - __uint_as_float(r[1] << 16), h[3] - __uint_as_float(r[1] & 0xffff0000u));
    return r;
}
// four values of a row of B from p on, n of them inside, in the form that second() needs
__device__ __forceinline__ raw4 factor4(const float* p, int n) { return n <= 0 ? raw4{0u, 0u, 0u, 0u} : load_part(p, n); }
__device__ __forceinline__ raw4 factor4(const bf16_t* p, int n) {
    raw2 r = {0u, 0u};
    if (n >= 4) r = *(const raw2_any*)p;
    else
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < n) r[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
    return raw4{r[0], r[1], r[0], r[1]};
}

constexpr int kWaves = 4;

// The sum over the waves' parts of k, and what follows from it for every wave: h for the second product, and h itself if kept
template <class T, int RT, int TT> struct Shared { f4 part[kWaves][RT * TT][64]; };
template <class T, int RT, int TT>
__device__ __forceinline__ void join(Shared<T, RT, TT>& sh, f4 (&acc)[RT][TT], raw4 (&h)[RT][TT], int rank, float scale, float* keep, const int64_t* tok, const bool* in) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < TT; ++t) sh.part[wave][r * TT + t][lane] = acc[r][t];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int i = r * TT + t;
            f4 v = (sh.part[0][i][lane] + sh.part[1][i][lane]) + (sh.part[2][i][lane] + sh.part[3][i][lane]);
            const int r0 = 16 * r + 4 * g;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r0 + j >= rank) v[j] = 0.f;                  // rows of A behind the rank were read from its last row
            if (keep && wave == i % kWaves && in[t]) {
                float* q = keep + tok[t] * rank + r0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (r0 + j < rank) q[j] = v[j];
            }
            h[r][t] = second<T>(v * scale);
        }
}

// Token rows.  A workgroup takes 16 TT tokens of a segment; its waves share the k of the first product (each takes every fourth
// 64 bytes of a row, so the four read 256 contiguous bytes) and the output channels of the second.  blockIdx.y splits the
// output channels where there are few tokens; each part then computes h for itself, from cache.
template <class T, int RT, int TT>
__global__ __launch_bounds__(64 * kWaves) void lora_rows_kernel(SegTable sg, k82_lora p) {
    constexpr int V = Vec<T>::N, K = 4 * V, U = RT * TT >= 8 ? 2 : 4;            // U: steps whose loads are in flight together
    __shared__ Shared<T, RT, TT> sh;
    const int s = seg_of(sg, blockIdx.x), k = sg.index[s];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    if (k < 0 && p.act == K82_ACT_NONE && p.base == p.y && !p.h) return;
    int64_t tok[TT];
    bool in[TT];
    const int row0 = ((int)blockIdx.x - sg.tile0[s]) * 16 * TT;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        const int i = row0 + 16 * t + col;
        in[t] = i < sg.len[s];
        tok[t] = sg.start[s] + min(i, sg.len[s] - 1);
    }
    f4 acc[RT][TT];
    raw4 h[RT][TT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < TT; ++t) { acc[r][t] = f4{0.f, 0.f, 0.f, 0.f}; h[r][t] = raw4{0u, 0u, 0u, 0u}; }
    if (k >= 0) {
        const T *a[RT], *x[TT];
#pragma unroll
        for (int r = 0; r < RT; ++r) a[r] = (const T*)p.a + ((int64_t)k * p.rank + min(16 * r + col, p.rank - 1)) * p.cin + g * V;
#pragma unroll
        for (int t = 0; t < TT; ++t) x[t] = (const T*)p.x + tok[t] * p.ldx + g * V;
        const int full = p.cin / K;
        auto steps = [&](int i0, auto n) {
            constexpr int n_ = decltype(n)::value;
            raw4 fa[n_][RT], fx[n_][TT];
#pragma unroll
            for (int i = 0; i < n_; ++i) {
                const int at = (i0 + i * kWaves) * K;
#pragma unroll
                for (int t = 0; t < TT; ++t) fx[i][t] = *(const raw4_any*)(x[t] + at);
#pragma unroll
                for (int r = 0; r < RT; ++r) fa[i][r] = *(const raw4_any*)(a[r] + at);
            }
#pragma unroll
            for (int i = 0; i < n_; ++i)
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int t = 0; t < TT; ++t) acc[r][t] = product<T>(fa[i][r], fx[i][t], acc[r][t]);
        };
        int i = wave;
        for (; i + (U - 1) * kWaves < full; i += U * kWaves) steps(i, std::integral_constant<int, U>());
        for (; i < full; i += kWaves) steps(i, std::integral_constant<int, 1>());
        if (i == full && p.cin % K) {                            // one wave: the end of the row, zeros behind it
            const int at = full * K, n = p.cin - at - g * V;
            raw4 fa[RT], fx[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) fx[t] = n > 0 ? load_part(x[t] + at, n) : raw4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int r = 0; r < RT; ++r) fa[r] = n > 0 ? load_part(a[r] + at, n) : raw4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int t = 0; t < TT; ++t) acc[r][t] = product<T>(fa[r], fx[t], acc[r][t]);
        }
        join<T, RT, TT>(sh, acc, h, p.rank, p.scale[k], blockIdx.y == 0 ? p.h : nullptr, tok, in);
    } else if (p.h && blockIdx.y == 0) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
            if (in[t])
                for (int r = 4 * wave + g; r < p.rank; r += 4 * kWaves) p.h[tok[t] * p.rank + r] = 0.f;
    }
    // Second product: V consecutive channels a lane (16 bytes of y), 4 V a block of the wave: the rows of B behind the 16 rows of
    // instruction j are the channels V (row / 4) + 4 j + row % 4.
    constexpr int J = V / 4;
    const T* b = (const T*)p.b + (int64_t)max(k, 0) * p.cout * p.rank;
    const int blocks = (p.cout + K - 1) / K;
    for (int blk = 2 * ((int)blockIdx.y * kWaves + wave); blk < blocks; blk += 2 * kWaves * gridDim.y) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int c0 = (blk + half) * K, mine = c0 + g * V, n = p.cout - mine;
            if (c0 >= p.cout) break;
            f4 d[TT][J];
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                raw4 v = {0u, 0u, 0u, 0u};
                if (p.base && n > 0) v = load_part((const T*)p.base + tok[t] * p.ldbase + mine, n);
                float f[V];
                Vec<T>::unpack(v, f);
#pragma unroll
                for (int j = 0; j < J; ++j) d[t][j] = f4{f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]};
            }
            if (k >= 0)
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const T* q = b + (int64_t)min(c0 + V * (col >> 2) + 4 * j + (col & 3), p.cout - 1) * p.rank + 4 * g;
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const raw4 f = factor4(q + 16 * r, p.rank - 16 * r - 4 * g);
#pragma unroll
                        for (int t = 0; t < TT; ++t) d[t][j] = product<T>(f, h[r][t], d[t][j]);
                    }
                }
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                float f[V];
#pragma unroll
                for (int j = 0; j < V; ++j) f[j] = d[t][j >> 2][j & 3];
                if (p.act == K82_ACT_GELU_NEW)
#pragma unroll
                    for (int j = 0; j < V; ++j) f[j] = op_gelu_new(f[j]);
                if (in[t] && n > 0) store_part((T*)p.y + tok[t] * p.ldy + mine, f, n);
            }
        }
    }
}

// Channel-first: the same products, TT consecutive tokens a lane (tile t of a lane's tokens is TT col + t), 16 TT tokens a
// workgroup, on the token grid of the tensor.  A tile that holds several segments is walked once for each.
template <int TT> __device__ __forceinline__ void load_tokens(float (&v)[TT], const float* p, int64_t t, int64_t lo, int64_t hi) {
    if (t >= lo && t + TT <= hi) {
        if constexpr (TT == 4) { const raw4 r = *(const raw4_f*)(p + t); for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(r[j]); }
        else { const f2_any r = *(const f2_any*)(p + t); v[0] = r[0]; v[1] = r[1]; }
        return;
    }
#pragma unroll
    for (int j = 0; j < TT; ++j) v[j] = t + j >= lo && t + j < hi ? p[t + j] : 0.f;
}
template <int RT, int TT>
__global__ __launch_bounds__(64 * kWaves) void lora_cols_kernel(SegTable sg, k82_lora p) {
    __shared__ Shared<float, RT, TT> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int first = sg.start[0];
    const int tile = first / (16 * TT) * (16 * TT) + (int)blockIdx.x * 16 * TT;
    const int64_t t0 = tile + TT * col;
    int s = place(sg.tile0, max(tile, first) - first);
    for (; s < sg.n && sg.start[s] < tile + 16 * TT; ++s) {
        const int k = sg.index[s];
        const int64_t lo = sg.start[s], hi = (int64_t)sg.start[s] + sg.len[s];
        if (k < 0 && p.act == K82_ACT_NONE && p.base == p.y && !p.h) continue;
        int64_t tok[TT];
        bool in[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) { tok[t] = t0 + t; in[t] = tok[t] >= lo && tok[t] < hi; }
        f4 acc[RT][TT];
        raw4 h[RT][TT];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < TT; ++t) { acc[r][t] = f4{0.f, 0.f, 0.f, 0.f}; h[r][t] = raw4{0u, 0u, 0u, 0u}; }
        if (k >= 0) {
            const float* a[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) a[r] = (const float*)p.a + ((int64_t)k * p.rank + min(16 * r + col, p.rank - 1)) * p.cin;
            auto step = [&](int c0, bool whole) {                // 16 channels: 4 g + i in instruction i
                float fx[4][TT];
                raw4 fa[RT];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = c0 + 4 * g + i;
                    if (whole || c < p.cin) load_tokens<TT>(fx[i], (const float*)p.x + (int64_t)c * p.ldx, t0, lo, hi);
                    else
#pragma unroll
                        for (int t = 0; t < TT; ++t) fx[i][t] = 0.f;
                }
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    fa[r] = whole ? *(const raw4_f*)(a[r] + c0 + 4 * g) : factor4(a[r] + c0 + 4 * g, p.cin - c0 - 4 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int t = 0; t < TT; ++t)
                            acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(fa[r][i]), fx[i][t], acc[r][t], 0, 0, 0);
            };
            const int full = p.cin / 16;
            int i = wave;
            for (; i < full; i += kWaves) step(16 * i, true);
            if (i == full && p.cin % 16) step(16 * i, false);
            join<float, RT, TT>(sh, acc, h, p.rank, p.scale[k], blockIdx.y == 0 ? p.h : nullptr, tok, in);
        } else if (p.h && blockIdx.y == 0) {
#pragma unroll
            for (int t = 0; t < TT; ++t)
                if (in[t])
                    for (int r = 4 * wave + g; r < p.rank; r += 4 * kWaves) p.h[tok[t] * p.rank + r] = 0.f;
        }
        const float* b = (const float*)p.b + (int64_t)max(k, 0) * p.cout * p.rank;
        const int blocks = (p.cout + 15) / 16;
        for (int blk = (int)blockIdx.y * kWaves + wave; blk < blocks; blk += kWaves * gridDim.y) {
            const int c0 = 16 * blk;
            float y[4][TT];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = c0 + 4 * g + i;
                if (p.base && c < p.cout) load_tokens<TT>(y[i], (const float*)p.base + (int64_t)c * p.ldbase, t0, lo, hi);
                else
#pragma unroll
                    for (int t = 0; t < TT; ++t) y[i][t] = 0.f;
            }
            f4 d[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) d[t] = f4{y[0][t], y[1][t], y[2][t], y[3][t]};
            if (k >= 0) {
                const float* q = b + (int64_t)min(c0 + col, p.cout - 1) * p.rank + 4 * g;
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const raw4 f = factor4(q + 16 * r, p.rank - 16 * r - 4 * g);
#pragma unroll
                    for (int t = 0; t < TT; ++t) d[t] = product<float>(f, h[r][t], d[t]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = c0 + 4 * g + i;
                if (c >= p.cout) continue;
                float* q = (float*)p.y + (int64_t)c * p.ldy + t0;
                float v[TT];
#pragma unroll
                for (int t = 0; t < TT; ++t) v[t] = p.act == K82_ACT_GELU_NEW ? op_gelu_new(d[t][i]) : d[t][i];
                if (in[0] && in[TT - 1]) {
                    if constexpr (TT == 4) *(raw4_f*)q = raw4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
                    else *(f2_any*)q = f2_any{v[0], v[1]};
                } else
#pragma unroll
                    for (int t = 0; t < TT; ++t)
                        if (in[t]) q[t] = v[t];
            }
        }
    }
}

// Backward.  dx = dx_base + s_k (dy B_k) A_k is the forward operator with B_k^T and A_k^T for A and B, and the h it keeps is
// g / s_k = dy B_k.  The transposed factors of the adapters in use are laid out here, side by side in the order of their index.
struct Used { int n, index[op::kSegs]; };
template <class T> __global__ __launch_bounds__(256) void lora_transpose_kernel(Used u, k82_lora_grad p, T* at, T* bt, float* scale) {
    __shared__ T tile[32][33];
    const int k = u.index[blockIdx.z], x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const bool is_b = blockIdx.x >= (unsigned)(p.cin + 31) / 32;
    const int c0 = 32 * (is_b ? (int)blockIdx.x - (p.cin + 31) / 32 : (int)blockIdx.x), r0 = 32 * blockIdx.y;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) scale[blockIdx.z] = p.scale[k];
    const int width = is_b ? p.cout : p.cin;
    const int64_t size = (int64_t)p.rank * width;
    for (int i = y; i < 32; i += 8) {                            // A: row r, B: row o
        const int row = (is_b ? c0 : r0) + i, c = (is_b ? r0 : c0) + x;
        if (row < (is_b ? width : p.rank) && c < (is_b ? p.rank : width))
            tile[i][x] = ((const T*)(is_b ? p.b : p.a))[k * size + (int64_t)row * (is_b ? p.rank : width) + c];
    }
    __syncthreads();
    for (int i = y; i < 32; i += 8) {
        const int row = (is_b ? r0 : c0) + i, c = (is_b ? c0 : r0) + x;
        if (row < (is_b ? p.rank : width) && c < (is_b ? width : p.rank))
            (is_b ? bt : at)[blockIdx.z * size + (int64_t)row * (is_b ? width : p.rank) + c] = tile[x][i];
    }
}

// 32 tokens x 8 channels a lane (bf16), transposed in registers: out[q] holds channel q of the lane's 8 tokens
__device__ __forceinline__ void transpose8(const raw4 (&in)[8], raw4 (&out)[8]) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            out[q][j] = __builtin_amdgcn_perm(in[2 * j + 1][q >> 1], in[2 * j][q >> 1], q & 1 ? 0x07060302u : 0x05040100u);
}
// 8 values of g in three bf16 parts: 24 bits, what a 32-bit sum of exact products deserves
__device__ __forceinline__ void split3(const float (&v)[8], raw4& hi, raw4& mid, raw4& lo) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a = v[2 * j], b = v[2 * j + 1];
        hi[j] = bf16_pair(a, b);
        a -= __uint_as_float(hi[j] << 16);
        b -= __uint_as_float(hi[j] & 0xffff0000u);
        mid[j] = bf16_pair(a, b);
        lo[j] = bf16_pair(a - __uint_as_float(mid[j] << 16), b - __uint_as_float(mid[j] & 0xffff0000u));
    }
}
// Sums over tokens: part[chunk][r][cin + cout] = s_k sum_t v_t[r] z_t[c] with (v, z) = (g / s_k, x) for the first cin channels
// and (h, dy) behind them.  A wave owns 128 channels of one of the two for all the tokens of a chunk.  The token axis is the
// k of the product: f32 takes it as it lies (4 tokens an instruction), bf16 through the transpose in registers.
template <class T, int RT>
__global__ __launch_bounds__(64 * kWaves) void lora_weight_kernel(RunTable rt, k82_lora_grad p, const float* gs, const float* scales, int used0, float* part) {
    constexpr int V = Vec<T>::N, M = 8;                          // 16 x 16 tiles along the channels
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int chunk = rt.chunk0[0] + (int)blockIdx.x, run = place(rt.chunk0, chunk);
    const int u0 = rt.run_cum[run] + (chunk - rt.chunk0[run]) * rt.rows, u1 = min(u0 + rt.rows, rt.run_cum[run + 1]);
    int slice = (int)blockIdx.y * kWaves + wave;
    const int nx = (p.cin + 127) / 128, ny = (p.cout + 127) / 128;
    if (slice >= nx + ny) return;
    const bool of_x = slice < nx;
    if (!of_x) slice -= nx;
    const T* z = (const T*)(of_x ? p.x : p.dy);
    const int64_t ld = of_x ? p.ldx : p.lddy;
    const int width = of_x ? p.cin : p.cout, c0 = 128 * slice;
    const float* v = of_x ? gs : p.h;
    f4 acc[M][RT];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[m][r] = f4{0.f, 0.f, 0.f, 0.f};
    int piece = place(rt.cum, u0);
    for (int u = u0; u < u1; ++piece) {                          // the pieces of a chunk, each a run of neighbouring tokens
        const int stop = min(u1, rt.cum[piece + 1]);
        const int64_t t0 = rt.start[piece] + (u - rt.cum[piece]);
        const int n = stop - u;
        u = stop;
        if constexpr (V == 8) {
            const int c = c0 + 8 * col, left = width - c;
            for (int i = 0; i < n; i += 32) {
                raw4 raw[8], zt[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int t = i + 8 * g + j;
                    raw[j] = raw4{0u, 0u, 0u, 0u};
                    if (t < n && left > 0) raw[j] = load_part(z + (t0 + t) * ld + c, left);
                }
                raw4 part3[RT][3];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    float w[8];
                    const int at = min(16 * r + col, p.rank - 1);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int t = i + 8 * g + j;
                        w[j] = t < n ? v[(t0 + t) * p.rank + at] : 0.f;
                    }
                    split3(w, part3[r][0], part3[r][1], part3[r][2]);
                }
                transpose8(raw, zt);
#pragma unroll
                for (int m = 0; m < 8; ++m)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int q = 2; q >= 0; --q) acc[m][r] = product<T>(zt[m], part3[r][q], acc[m][r]);
            }
        } else {
            for (int i = 0; i < n; i += 4) {
                const int t = i + g;
                raw4 raw[2];
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const int c = c0 + 64 * m + 4 * col;
                    raw[m] = raw4{0u, 0u, 0u, 0u};
                    if (t < n && c < width) raw[m] = load_part(z + (t0 + t) * ld + c, width - c);
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const float w = t < n ? v[(t0 + t) * p.rank + min(16 * r + col, p.rank - 1)] : 0.f;
#pragma unroll
                    for (int m = 0; m < 8; ++m)
                        acc[m][r] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(raw[m >> 2][m & 3]), w, acc[m][r], 0, 0, 0);
                }
            }
        }
    }
    // row 4 g + i of tile m is the channel 8 (4 g + i) + m (bf16) or 64 (m / 4) + 4 (4 g + i) + m % 4 (f32)
    const float scale = scales[used0 + run];
    float* out = part + (int64_t)chunk * p.rank * (p.cin + p.cout) + (of_x ? 0 : p.cin);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        if (16 * r + col >= p.rank) continue;
        float* q = out + (int64_t)(16 * r + col) * (p.cin + p.cout);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int m = 0; m < M; m += 4) {
                const int c = c0 + (V == 8 ? 8 * (4 * g + i) + m : 16 * m + 4 * (4 * g + i));
                const float f[4] = {acc[m][r][i] * scale, acc[m + 1][r][i] * scale, acc[m + 2][r][i] * scale, acc[m + 3][r][i] * scale};
                if (c < width) store_part(q + c, f, width - c);
            }
    }
}
// da, db: the chunks of an adapter in order
__global__ __launch_bounds__(256) void lora_reduce_kernel(ReduceTable rt, int cin, int cout, int rank, const float* part, float* da, float* db) {
    const int c = (int)blockIdx.x * 256 + (int)threadIdx.x, r = blockIdx.y, k = blockIdx.z;
    if (c >= cin + cout) return;
    float s = 0.f;
    for (int i = rt.first[k]; i < rt.first[k + 1]; ++i) s += part[((int64_t)i * rank + r) * (cin + cout) + c];
    if (c < cin) da[((int64_t)(rt.base + k) * rank + r) * cin + c] = s;
    else db[((int64_t)(rt.base + k) * cout + (c - cin)) * rank + r] = s;
}

template <class F> hipError_t by_rank(int rank, F&& f) {
    if (rank <= 16) return f(std::integral_constant<int, 1>());
    if (rank <= 32) return f(std::integral_constant<int, 2>());
    if (rank <= 64) return f(std::integral_constant<int, 4>());
    return f(std::integral_constant<int, 8>());
}
// parts of the output channels: until there are two workgroups a CU, at least 64 channels a wave
int parts(int tiles, int cout) { return std::max(1, std::min((cout + 255) / 256, 512 / std::max(1, tiles))); }

template <class T> hipError_t forward(const k82_lora& p, const std::vector<op::Seg>& segs, hipStream_t st) {
    return by_rank(p.rank, [&](auto rt) -> hipError_t {
        constexpr int RT = decltype(rt)::value, TT = RT == 4 ? 4 : 2;
        if constexpr (std::is_same<T, float>::value)
            if (p.layout == K82_COLS) {
                for (const SegTable& t : op::tables(segs, 1)) {
                    const int first = t.start[0], last = first + t.tile0[t.n] - 1, tiles = last / 32 - first / 32 + 1;
                    OP_TRY(op::run(lora_cols_kernel<RT, 2>, dim3(tiles, parts(tiles, p.cout)), dim3(64 * kWaves), 0, st, t, p));
                }
                return hipSuccess;
            }
        for (const SegTable& t : op::tables(segs, 16 * TT)) {
            const int tiles = t.tile0[t.n];
            OP_TRY(op::run(lora_rows_kernel<T, RT, TT>, dim3(tiles, parts(tiles, p.cout)), dim3(64 * kWaves), 0, st, t, p));
        }
        return hipSuccess;
    });
}

// tokens of a chunk of the weight's gradient: two workgroups a CU once there are tokens for them
int chunk_rows(const k82_lora_grad& p, int64_t tokens) {
    const int64_t slices = ((p.cin + 127) / 128 + (p.cout + 127) / 128 + kWaves - 1) / kWaves;
    const int64_t chunks = std::max<int64_t>(1, 512 / slices);
    return (int)std::max<int64_t>(64, ((tokens + chunks - 1) / chunks + 31) / 32 * 32);
}
struct Layout { int64_t g, at, bt, scale, part, end; };         // bytes
Layout layout(const k82_lora_grad& p, const k82_segments& s) {
    const int64_t size = p.dtype == K82_F32 ? 4 : 2, used = std::min<int64_t>(s.n, p.adapters), all = (int64_t)p.cin + p.cout;
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    Layout l;
    l.g = 0;
    l.at = up(l.g + p.tokens * p.rank * 4);
    l.bt = up(l.at + used * p.rank * p.cin * size);
    l.scale = up(l.bt + used * p.rank * p.cout * size);
    l.part = up(l.scale + used * 4);
    l.end = l.part + op::most_chunks(s, p.adapters, chunk_rows(p, op::covered(s))) * p.rank * all * 4;
    return l;
}
template <class T> hipError_t backward(const k82_lora_grad& p, const k82_segments& s, void* ws, hipStream_t st) {
    const Layout l = layout(p, s);
    const op::RunPlan plan = op::runs(s, p.adapters, chunk_rows(p, op::covered(s)));
    char* w = (char*)ws;
    float *g = (float*)(w + l.g), *scale = (float*)(w + l.scale), *part = (float*)(w + l.part);
    T *at = (T*)(w + l.at), *bt = (T*)(w + l.bt);
    // the adapters in use, numbered in the order of their index
    std::vector<int> used, number(p.adapters, -1), first;
    for (const RunTable& t : plan.tables) {
        first.push_back((int)used.size());
        for (int i = 0; i < t.runs; ++i) {
            if (number[t.index[i]] < 0) { number[t.index[i]] = (int)used.size(); used.push_back(t.index[i]); }
            else first.back() = number[t.index[i]];              // a run that the table before began
        }
    }
    const int64_t factor = (int64_t)p.rank;
    for (size_t i = 0; i < used.size(); i += op::kSegs) {
        Used u;
        u.n = (int)std::min<size_t>(op::kSegs, used.size() - i);
        std::copy_n(used.begin() + i, u.n, u.index);
        OP_TRY(op::run(lora_transpose_kernel<T>, dim3((p.cin + 31) / 32 + (p.cout + 31) / 32, (p.rank + 31) / 32, u.n), dim3(256), 0, st, u, p,
                       at + i * factor * p.cin, bt + i * factor * p.cout, scale + i));
    }
    std::vector<op::Seg> segs = op::merged(s);
    for (op::Seg& v : segs)
        if (v.index >= 0) v.index = number[v.index];
    const k82_lora f{p.dtype, K82_ROWS, K82_ACT_NONE, p.cout, p.cin, p.rank, (int)used.size(), p.tokens, p.dy, p.lddy,
                     p.dx_base, p.lddx_base, p.dx, p.lddx, bt, at, scale, g};
    OP_TRY(forward<T>(f, segs, st));
    const int slices = ((p.cin + 127) / 128 + (p.cout + 127) / 128 + kWaves - 1) / kWaves;
    for (size_t i = 0; i < plan.tables.size(); ++i) {
        const RunTable& t = plan.tables[i];
        OP_TRY(by_rank(p.rank, [&](auto rt) {
            return op::run(lora_weight_kernel<T, decltype(rt)::value>, dim3(t.chunk0[t.runs] - t.chunk0[0], slices), dim3(64 * kWaves), 0, st, t, p,
                           (const float*)g, (const float*)scale, first[i], part);
        }));
    }
    for (const ReduceTable& t : plan.reduce)
        OP_TRY(op::run(lora_reduce_kernel, dim3((p.cin + p.cout + 255) / 256, p.rank, t.n), dim3(256), 0, st, t, p.cin, p.cout, p.rank,
                       (const float*)part, p.da, p.db));
    return hipSuccess;
}
}  // namespace

namespace op {
int64_t workspace(const k82_lora_grad& p, const k82_segments& s) { return layout(p, s).end; }
hipError_t launch(const k82_lora& p, const k82_segments& s, hipStream_t st) {
    return p.dtype == K82_F32 ? forward<float>(p, merged(s), st) : forward<bf16_t>(p, merged(s), st);
}
hipError_t launch(const k82_lora_grad& p, const k82_segments& s, void* ws, hipStream_t st) {
    return p.dtype == K82_F32 ? backward<float>(p, s, ws, st) : backward<bf16_t>(p, s, ws, st);
}
}  // namespace op
