// Layer norm with a gain / offset per segment: z = x + res, y = (z - mean) rstd gain_k + offset_k, and its gradients.
// All forms are bound by memory: a row is read once into registers, the mean and then the centred square sum are taken from
// there (the variance never comes from a difference of large sums), and the result leaves from the same registers.
#include "operators.h"

#include <algorithm>

namespace {
using op::ReduceTable;
using op::RunTable;
using op::SegTable;

// A row of c channels is held by W waves, NV 16-byte vectors a lane: NV <= 16 bytes / element, so at most 16 values a lane.
constexpr int kRowMax = 16 * 1024;             // channels that fit the registers of 16 waves
constexpr int kGradRowMax = 8 * 1024;          // ... beside the sums and the gain of the backward pass
template <int W> constexpr int kThreads = W == 1 ? 256 : 64 * W;      // W == 1: four rows side by side

// Sum over the W waves of a row.  `sh` is a buffer of this one reduction: written, barrier, read; it is written again only
// behind another barrier that the caller's next reduction brings.
template <int W> __device__ __forceinline__ float row_total(float v, float* sh) {
    v = wave_total(v);
    if constexpr (W == 1) return v;
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += sh[i];
    return s;
}

template <class T, int W, int NV>
__global__ __launch_bounds__(kThreads<W>) void norm_rows_kernel(SegTable sg, k82_layernorm p, int tile) {
    constexpr int N = Vec<T>::N, R = W == 1 ? 4 : 1;
    __shared__ float sh[2][W];
    const int lane = W == 1 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
    const int wave = W == 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0;
    const int seg = seg_of(sg, blockIdx.x), begin = ((int)blockIdx.x - sg.tile0[seg]) * tile;
    const int end = sg.start[seg] + min(sg.len[seg], begin + tile);
    int t = sg.start[seg] + begin + wave;
    float g[NV][N], o[NV][N];
    int left[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (lane + i * 64 * W) * N;
        left[i] = p.c - c;                                       // channels from this vector on
        raw4 a = {0u, 0u, 0u, 0u}, b = a;
        if (left[i] > 0) {
            a = load_part((const T*)p.gain + (int64_t)sg.index[seg] * p.c + c, left[i]);
            b = load_part((const T*)p.offset + (int64_t)sg.index[seg] * p.c + c, left[i]);
        }
        Vec<T>::unpack(a, g[i]);
        Vec<T>::unpack(b, o[i]);
    }
    auto fetch = [&](int64_t row, raw4* rx, raw4* rr) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (lane + i * 64 * W) * N;
            if (left[i] > 0) {
                rx[i] = load_part((const T*)p.x + row * p.ldx + c, left[i]);
                if (p.res) rr[i] = load_part((const T*)p.res + row * p.ldres + c, left[i]);
            }
        }
    };
    raw4 rx[NV], rr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) rx[i] = rr[i] = raw4{0u, 0u, 0u, 0u};
    if (t < end) fetch(t, rx, rr);
    for (; t < end; t += R) {
        float z[NV][N];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float r[N];
            Vec<T>::unpack(rx[i], z[i]);
            Vec<T>::unpack(rr[i], r);
#pragma unroll
            for (int j = 0; j < N; ++j) { z[i][j] += r[j]; s += z[i][j]; }
        }
        if (t + R < end) fetch(t + R, rx, rr);                   // the next row is on its way while this one is summed
        const float mean = row_total<W>(s, sh[0]) / p.c;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < N; ++j) z[i][j] -= mean;
            if (left[i] < N) {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (j >= left[i]) z[i][j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) q = fmaf(z[i][j], z[i][j], q);
        }
        const float rstd = 1.0f / sqrtf(row_total<W>(q, sh[1]) / p.c + p.eps);
        if (p.mean && lane == 0) { p.mean[t] = mean; p.rstd[t] = rstd; }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float y[N];
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] = fmaf(z[i][j] * rstd, g[i][j], o[i][j]);
            if (left[i] > 0) store_part((T*)p.y + (int64_t)t * p.ldy + (lane + i * 64 * W) * N, y, left[i]);
        }
    }
}

// Channel-first rows (the engine's layout).  A workgroup of NW waves holds 4 Q tokens: a lane has four of them (16 bytes) of
// every STEP-th channel, a wave's load covers 64 / Q channels.  Tiles lie on the token grid of the tensor, not of the
// sentences: rows start on lines and a batch of short sentences fills its tiles; the gain row is picked by token where a tile
// holds several sentences.  The shape goes by the channel count alone, so a token's bits do not depend on its batch.
// 32 tokens are the 128 bytes of a line: 16411 x 768 with a residual 47 us (3.2 TB/s; token rows: 34 us); 64 tokens 51 us and
// 16 tokens 50 to 56 us.  All of a tile is loaded, then all of it stored, which two workgroups on a CU overlap only in part.
constexpr int kColsMax = 4096;                 // channels that fit
template <int Q, int NW, int NV> __global__ __launch_bounds__(64 * NW) void norm_cols_kernel(SegTable sg, k82_layernorm p) {
    constexpr int TOK = 4 * Q, STEP = NW * 64 / Q;               // tokens of a tile, channels of a round
    __shared__ float4 red[2][NW][Q];
    __shared__ int kind[TOK];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quad = lane & (Q - 1);
    const int first = sg.start[0], end = first + sg.tile0[sg.n];
    const int t0 = (first & ~(TOK - 1)) + (int)blockIdx.x * TOK + 4 * quad, c0 = 64 / Q * wave + lane / Q;
    const bool whole = t0 >= first && t0 + 4 <= end;             // (what is loaded there; skipped tokens are not stored)
    if (threadIdx.x < TOK) {
        const int t = min(max((first & ~(TOK - 1)) + (int)blockIdx.x * TOK + (int)threadIdx.x, first), end - 1) - first;
        int s = 0;
        for (int step = op::kSegs / 2; step > 0; step >>= 1)     // last segment that starts at or before t
            if (s + step < sg.n && sg.tile0[s + step] <= t) s += step;
        kind[threadIdx.x] = sg.index[s];
    }
    auto fetch = [&](const void* q, int64_t ld, int c) -> float4 {
        const float* v = (const float*)q + (int64_t)c * ld + t0;
        if (whole) { const raw4 r = *(const raw4_f*)v; return make_float4(__uint_as_float(r[0]), __uint_as_float(r[1]), __uint_as_float(r[2]), __uint_as_float(r[3])); }
        auto at = [&](int j) { return t0 + j >= first && t0 + j < end ? v[j] : 0.f; };
        return make_float4(at(0), at(1), at(2), at(3));
    };
    float4 z[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) z[i] = c0 + STEP * i < p.c ? fetch(p.x, p.ldx, c0 + STEP * i) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.res) {
        float4 r[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) r[i] = c0 + STEP * i < p.c ? fetch(p.res, p.ldres, c0 + STEP * i) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i) z[i] = make_float4(z[i].x + r[i].x, z[i].y + r[i].y, z[i].z + r[i].z, z[i].w + r[i].w);
    }
    // sum over the channels: the lane's own, the four of a wave, the 16 waves
    auto total = [&](float4 v, float4 (&buf)[NW][Q]) -> float4 {
        float a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int m = Q; m < 64; m *= 2)
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] += __shfl_xor(a[j], m, 64);
        if (lane < Q) buf[wave][quad] = make_float4(a[0], a[1], a[2], a[3]);
        __syncthreads();
        float4 s = buf[0][quad];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            const float4 b = buf[w][quad];
            s = make_float4(s.x + b.x, s.y + b.y, s.z + b.z, s.w + b.w);
        }
        return s;
    };
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) s = make_float4(s.x + z[i].x, s.y + z[i].y, s.z + z[i].z, s.w + z[i].w);
    s = total(s, red[0]);
    const float4 mean = make_float4(s.x / p.c, s.y / p.c, s.z / p.c, s.w / p.c);
    float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (c0 + STEP * i < p.c) {
            z[i] = make_float4(z[i].x - mean.x, z[i].y - mean.y, z[i].z - mean.z, z[i].w - mean.w);
            q = make_float4(fmaf(z[i].x, z[i].x, q.x), fmaf(z[i].y, z[i].y, q.y), fmaf(z[i].z, z[i].z, q.z), fmaf(z[i].w, z[i].w, q.w));
        }
    }
    q = total(q, red[1]);
    const float4 rstd = make_float4(1.0f / sqrtf(q.x / p.c + p.eps), 1.0f / sqrtf(q.y / p.c + p.eps),
                                    1.0f / sqrtf(q.z / p.c + p.eps), 1.0f / sqrtf(q.w / p.c + p.eps));
    const int k0 = kind[4 * quad], k1 = kind[4 * quad + 1], k2 = kind[4 * quad + 2], k3 = kind[4 * quad + 3];
    const bool stored[4] = {t0 >= first && t0 < end && k0 >= 0, t0 + 1 >= first && t0 + 1 < end && k1 >= 0,
                            t0 + 2 >= first && t0 + 2 < end && k2 >= 0, t0 + 3 >= first && t0 + 3 < end && k3 >= 0};
    const bool all4 = stored[0] && stored[1] && stored[2] && stored[3];
    auto store = [&](float* v, float4 y) {
        if (all4) { *(raw4_f*)v = raw4{__float_as_uint(y.x), __float_as_uint(y.y), __float_as_uint(y.z), __float_as_uint(y.w)}; return; }
        const float a[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (stored[j]) v[j] = a[j];
    };
    if (p.mean && c0 == 0) { store(p.mean + t0, mean); store(p.rstd + t0, rstd); }
    const float *gain = (const float*)p.gain, *offset = (const float*)p.offset;
    const bool uniform = __all(k0 == kind[0] && k1 == kind[0] && k2 == kind[0] && k3 == kind[0]);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + STEP * i;
        if (c >= p.c) continue;
        float4 g, o;
        const int64_t at = (int64_t)max(k0, 0) * p.c + c;
        g.x = gain[at]; o.x = offset[at];
        if (uniform) {
            g = make_float4(g.x, g.x, g.x, g.x);
            o = make_float4(o.x, o.x, o.x, o.x);
        } else {
            const int64_t a1 = (int64_t)max(k1, 0) * p.c + c, a2 = (int64_t)max(k2, 0) * p.c + c, a3 = (int64_t)max(k3, 0) * p.c + c;
            g = make_float4(g.x, gain[a1], gain[a2], gain[a3]);
            o = make_float4(o.x, offset[a1], offset[a2], offset[a3]);
        }
        store((float*)p.y + (int64_t)c * p.ldy + t0, make_float4(fmaf(z[i].x * rstd.x, g.x, o.x), fmaf(z[i].y * rstd.y, g.y, o.y),
                                                                 fmaf(z[i].z * rstd.z, g.z, o.z), fmaf(z[i].w * rstd.w, g.w, o.w)));
    }
}

template <int N> __device__ __forceinline__ float block_total(float v, float (&sh)[N]) {    // 64 N threads
    v = wave_total(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += sh[i];
    return s;
}

// Rows that no registers hold: one workgroup per token, the row read three times.
template <class T>
__global__ __launch_bounds__(256) void norm_token_kernel(SegTable sg, k82_layernorm p, int64_t xt, int64_t xc, int64_t rt, int64_t rc, int64_t yt, int64_t yc) {
    __shared__ float sh[4];
    const int s = seg_of(sg, blockIdx.x), k = sg.index[s];
    const int64_t t = sg.start[s] + ((int)blockIdx.x - sg.tile0[s]);
    const T *x = (const T*)p.x + t * xt, *res = p.res ? (const T*)p.res + t * rt : nullptr;
    auto z = [&](int c) { return to_f(x[c * xc]) + (res ? to_f(res[c * rc]) : 0.f); };
    float v = 0.f;
    for (int c = threadIdx.x; c < p.c; c += 256) v += z(c);
    const float mean = block_total(v, sh) / p.c;
    v = 0.f;
    for (int c = threadIdx.x; c < p.c; c += 256) { const float d = z(c) - mean; v = fmaf(d, d, v); }
    const float rstd = 1.0f / sqrtf(block_total(v, sh) / p.c + p.eps);
    if (p.mean && threadIdx.x == 0) { p.mean[t] = mean; p.rstd[t] = rstd; }
    const T *g = (const T*)p.gain + (int64_t)k * p.c, *o = (const T*)p.offset + (int64_t)k * p.c;
    for (int c = threadIdx.x; c < p.c; c += 256) put((T*)p.y + t * yt + c * yc, fmaf((z(c) - mean) * rstd, to_f(g[c]), to_f(o[c])));
}

// Backward: one pass over x, res and dy.  A workgroup takes a chunk of the tokens of one gain; a lane owns its channels for
// the whole chunk, so dy xh and dy are summed in its registers and leave once, as the chunk's partial sums.
// SPLIT (rows that no registers hold): the two row means come from `sums`, blockIdx.y picks 1024 channels.
template <class T, int W, int NV, bool SPLIT>
__global__ __launch_bounds__(kThreads<W>) void norm_grad_kernel(RunTable rt, k82_layernorm_grad p, const float2* sums, float* part) {
    constexpr int N = Vec<T>::N, R = W == 1 ? 4 : 1;
    __shared__ float sh[2][2][W];
    __shared__ float joint[W == 1 ? 4 * 64 * NV * N : 1];
    const int lane = W == 1 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
    const int wave = W == 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0;
    const int chunk = rt.chunk0[0] + (int)blockIdx.x, run = place(rt.chunk0, chunk);
    const int u0 = rt.run_cum[run] + (chunk - rt.chunk0[run]) * rt.rows, u1 = min(u0 + rt.rows, rt.run_cum[run + 1]);
    const int c0 = SPLIT ? (int)blockIdx.y * 1024 : 0;
    float g[NV][N], ag[NV][N], ab[NV][N];
    int left[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + (lane + i * 64 * W) * N;
        left[i] = p.c - c;
        raw4 a = {0u, 0u, 0u, 0u};
        if (left[i] > 0) a = load_part((const T*)p.gain + (int64_t)rt.index[run] * p.c + c, left[i]);
        Vec<T>::unpack(a, g[i]);
#pragma unroll
        for (int j = 0; j < N; ++j) ag[i][j] = ab[i][j] = 0.f;
    }
    int u = u0 + wave, piece = place(rt.cum, min(u, u1 - 1));
    raw4 rx[NV], rr[NV], rd[NV];
    float mean = 0.f, rstd = 0.f;
    float2 given = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) rx[i] = rr[i] = rd[i] = raw4{0u, 0u, 0u, 0u};
    int64_t t = 0;
    auto fetch = [&]() {                                         // row u: piece only moves forward
        while (u >= rt.cum[piece + 1]) ++piece;
        t = rt.start[piece] + (u - rt.cum[piece]);
        mean = p.mean[t];
        rstd = p.rstd[t];
        if constexpr (SPLIT) given = sums[t];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = c0 + (lane + i * 64 * W) * N;
            if (left[i] > 0) {
                rx[i] = load_part((const T*)p.x + t * p.ldx + c, left[i]);
                rd[i] = load_part((const T*)p.dy + t * p.lddy + c, left[i]);
                if (p.res) rr[i] = load_part((const T*)p.res + t * p.ldres + c, left[i]);
            }
        }
    };
    if (u < u1) fetch();
    int flip = 0;
    while (u < u1) {
        float xh[NV][N], w[NV][N];
        float s1 = 0.f, s2 = 0.f;
        const float r = rstd, m = mean;
        const float2 known = given;
        const int64_t row = t;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float res[N];
            Vec<T>::unpack(rx[i], xh[i]);
            Vec<T>::unpack(rr[i], res);
            Vec<T>::unpack(rd[i], w[i]);
#pragma unroll
            for (int j = 0; j < N; ++j) xh[i][j] = (xh[i][j] + res[j] - m) * r;
            if (left[i] < N) {                                   // channels behind the row add nothing, not 0 times an infinity
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (j >= left[i]) xh[i][j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                ag[i][j] = fmaf(w[i][j], xh[i][j], ag[i][j]);
                ab[i][j] += w[i][j];
                w[i][j] *= g[i][j];
                s1 += w[i][j];
                s2 = fmaf(w[i][j], xh[i][j], s2);
            }
        }
        u += R;
        if (u < u1) fetch();                                     // the next row is on its way while this one is summed
        if constexpr (SPLIT) {
            s1 = known.x;
            s2 = known.y;
        } else {
            s1 = wave_total(s1);
            s2 = wave_total(s2);
            if constexpr (W > 1) {                               // one barrier a row: two buffers in turn
                if ((threadIdx.x & 63) == 0) { sh[flip][0][threadIdx.x >> 6] = s1; sh[flip][1][threadIdx.x >> 6] = s2; }
                __syncthreads();
                s1 = s2 = 0.f;
#pragma unroll
                for (int k = 0; k < W; ++k) { s1 += sh[flip][0][k]; s2 += sh[flip][1][k]; }
                flip ^= 1;
            }
            s1 /= p.c;
            s2 /= p.c;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < N; ++j) w[i][j] = r * (w[i][j] - s1 - xh[i][j] * s2);
            if (left[i] > 0) store_part((T*)p.dx + row * p.lddx + c0 + (lane + i * 64 * W) * N, w[i], left[i]);
        }
    }
    float* out = part + (int64_t)chunk * 2 * p.c + c0;
    if constexpr (W == 1) {                                      // the four waves of a chunk, in order
        const int width = min(p.c - c0, 64 * NV * N);
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
            if (pass) __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j) joint[(wave * NV * 64 + i * 64 + lane) * N + j] = pass ? ab[i][j] : ag[i][j];
            __syncthreads();
            for (int c = threadIdx.x; c < width; c += 256)
                out[(int64_t)pass * p.c + c] = (joint[c] + joint[64 * NV * N + c]) + (joint[2 * 64 * NV * N + c] + joint[3 * 64 * NV * N + c]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (left[i] > 0) {
                const int c = (lane + i * 64 * W) * N;
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (j < left[i]) { out[c + j] = ag[i][j]; out[p.c + c + j] = ab[i][j]; }
            }
    }
}
// dgain, doffset: 64 columns a workgroup, 16 waves take every 16th chunk, their sums in order
__global__ __launch_bounds__(1024) void norm_reduce_kernel(ReduceTable rt, int c, const float* part, float* dgain, float* doffset) {
    __shared__ float sh[16][64];
    const int col = (int)blockIdx.x * 64 + ((int)threadIdx.x & 63), wave = threadIdx.x >> 6, k = blockIdx.y;
    float s = 0.f;
    if (col < 2 * c)
        for (int i = rt.first[k] + wave; i < rt.first[k + 1]; i += 16) s += part[(int64_t)i * 2 * c + col];
    sh[wave][threadIdx.x & 63] = s;
    __syncthreads();
    if (wave == 0 && col < 2 * c) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += sh[i][threadIdx.x];
        (col < c ? dgain + col : doffset + (col - c))[(int64_t)(rt.base + k) * c] = s;
    }
}
// the two row means of the backward pass, for rows that no registers hold
template <class T> __global__ __launch_bounds__(256) void norm_grad_sums_kernel(SegTable sg, k82_layernorm_grad p, float2* sums) {
    __shared__ float sh[4];
    const int s = seg_of(sg, blockIdx.x), k = sg.index[s];
    const int64_t t = sg.start[s] + ((int)blockIdx.x - sg.tile0[s]);
    const T *x = (const T*)p.x + t * p.ldx, *res = p.res ? (const T*)p.res + t * p.ldres : nullptr, *dy = (const T*)p.dy + t * p.lddy;
    const T* g = (const T*)p.gain + (int64_t)k * p.c;
    const float mean = p.mean[t], rstd = p.rstd[t];
    float v = 0.f, w = 0.f;
    for (int c = threadIdx.x; c < p.c; c += 256) {
        const float xh = (to_f(x[c]) + (res ? to_f(res[c]) : 0.f) - mean) * rstd, u = to_f(dy[c]) * to_f(g[c]);
        v += u;
        w = fmaf(u, xh, w);
    }
    v = block_total(v, sh) / p.c;
    w = block_total(w, sh) / p.c;
    if (threadIdx.x == 0) sums[t] = make_float2(v, w);
}

// The fewest waves whose registers hold a row, and the vectors a lane needs: calls f<W, NV>().
template <class T, int MAX, class F> hipError_t by_width(int c, F&& f) {
    constexpr int N = Vec<T>::N;
    const int vectors = (c + N - 1) / N;
    auto with = [&](auto w) -> hipError_t {
        constexpr int W = decltype(w)::value, M = std::min(16, MAX / (64 * W)) / N;
        const int nv = (vectors + 64 * W - 1) / (64 * W);
        if (nv <= 1) return f(w, std::integral_constant<int, 1>());
        if (nv == 2) return f(w, std::integral_constant<int, std::min(2, M)>());
        if (nv == 3) return f(w, std::integral_constant<int, std::min(3, M)>());
        return f(w, std::integral_constant<int, M>());
    };
    if (c <= 1024) return with(std::integral_constant<int, 1>());
    if (c <= 4096) return with(std::integral_constant<int, 4>());
    return with(std::integral_constant<int, 16>());
}

template <class T> hipError_t forward(const k82_layernorm& p, const k82_segments& s, hipStream_t st) {
    const bool cols = p.layout == K82_COLS;
    if (cols && p.c <= kColsMax) {
        for (const SegTable& t : op::tables(op::merged(s, true), 1)) {
            const int tokens = t.tile0[t.n];
            auto go = [&](auto q, auto w, auto v) {
                constexpr int Q = decltype(q)::value, NW = decltype(w)::value;
                const int tiles = (t.start[0] + tokens - 1) / (4 * Q) - t.start[0] / (4 * Q) + 1;
                return op::run(norm_cols_kernel<Q, NW, decltype(v)::value>, dim3(tiles), dim3(64 * NW), 0, st, t, p);
            };
            const std::integral_constant<int, 12> v12; const std::integral_constant<int, 2> q2; const std::integral_constant<int, 4> q4;
            const std::integral_constant<int, 8> q8; const std::integral_constant<int, 16> w16;
            OP_TRY(p.c <= 256 ? go(q8, q8, q4) : p.c <= 512 ? go(q8, q8, q8) : p.c <= 768 ? go(q8, q8, v12) :
                   p.c <= 1536 ? go(q8, w16, v12) : p.c <= 2048 ? go(q4, w16, q8) : go(q2, w16, q8));
        }
        return hipSuccess;
    }
    const std::vector<op::Seg> segs = op::merged(s);
    if (cols || p.c > kRowMax) {
        for (const SegTable& t : op::tables(segs, 1))
            OP_TRY(op::run(norm_token_kernel<T>, dim3(t.tile0[t.n]), dim3(256), 0, st, t, p, cols ? 1 : p.ldx, cols ? p.ldx : 1,
                           cols ? 1 : p.ldres, cols ? p.ldres : 1, cols ? 1 : p.ldy, cols ? p.ldy : 1));
        return hipSuccess;
    }
    return by_width<T, kRowMax>(p.c, [&](auto w, auto nv) -> hipError_t {
        constexpr int W = decltype(w)::value, R = W == 1 ? 4 : 1;
        // rows behind each other in a workgroup share the gain's registers, once there are rows for every CU (8 rather than 4 of
        // the widest where 1024 threads for every four would reach the 2^32 that a launch cannot hold)
        const int64_t tokens = op::covered(s), most = W == 16 && tokens >= 1 << 23 ? 8 : 4;
        const int tile = R * (int)std::max<int64_t>(1, std::min(most, tokens / (R * 2048)));
        for (const SegTable& t : op::tables(segs, tile))
            OP_TRY(op::run(norm_rows_kernel<T, W, decltype(nv)::value>, dim3(t.tile0[t.n]), dim3(kThreads<W>), 0, st, t, p, tile));
        return hipSuccess;
    });
}

// Tokens of a chunk: one workgroup for every place on the 256 CUs once there are tokens for them (the registers leave
// three of 256 threads to a CU; 131072 x 768 bf16 with a residual: 768 chunks 172 us, 1024 186 us, 512 185 us).
int chunk_rows(int c, int64_t tokens) {
    const int least = c <= 1024 || c > kGradRowMax ? 16 : c <= 4096 ? 8 : 4;
    const int64_t most = c <= 4096 || c > kGradRowMax ? 768 : 512;
    return (int)std::max<int64_t>(least, ((tokens + most - 1) / most + 3) / 4 * 4);
}
template <class T> hipError_t backward(const k82_layernorm_grad& p, const k82_segments& s, void* ws, hipStream_t st) {
    const op::RunPlan plan = op::runs(s, p.gains, chunk_rows(p.c, op::covered(s)));
    float* part = (float*)ws;
    float2* sums = nullptr;
    if (p.c > kGradRowMax) {
        sums = (float2*)ws;
        part = (float*)(sums + p.tokens);
        for (const SegTable& t : op::tables(op::merged(s), 1))
            OP_TRY(op::run(norm_grad_sums_kernel<T>, dim3(t.tile0[t.n]), dim3(256), 0, st, t, p, sums));
    }
    for (const RunTable& t : plan.tables) {
        const int chunks = t.chunk0[t.runs] - t.chunk0[0];
        if (sums) {
            OP_TRY(op::run(norm_grad_kernel<T, 1, 16 / Vec<T>::N, true>, dim3(chunks, (p.c + 1023) / 1024), dim3(256), 0, st, t, p, (const float2*)sums, part));
        } else {
            OP_TRY(by_width<T, kGradRowMax>(p.c, [&](auto w, auto nv) {
                constexpr int W = decltype(w)::value;
                return op::run(norm_grad_kernel<T, W, decltype(nv)::value, false>, dim3(chunks), dim3(kThreads<W>), 0, st, t, p, (const float2*)nullptr, part);
            }));
        }
    }
    for (const ReduceTable& t : plan.reduce)
        OP_TRY(op::run(norm_reduce_kernel, dim3((2 * p.c + 63) / 64, t.n), dim3(1024), 0, st, t, p.c, (const float*)part, p.dgain, p.doffset));
    return hipSuccess;
}
}  // namespace

namespace op {
int64_t workspace(const k82_layernorm_grad& p, const k82_segments& s) {
    return (p.c > kGradRowMax ? p.tokens * 8 : 0) + most_chunks(s, p.gains, chunk_rows(p.c, covered(s))) * 2 * p.c * 4;
}
hipError_t launch(const k82_layernorm& p, const k82_segments& s, hipStream_t st) {
    return p.dtype == K82_F32 ? forward<float>(p, s, st) : forward<bf16_t>(p, s, st);
}
hipError_t launch(const k82_layernorm_grad& p, const k82_segments& s, void* ws, hipStream_t st) {
    return p.dtype == K82_F32 ? backward<float>(p, s, ws, st) : backward<bf16_t>(p, s, ws, st);
}
}  // namespace op
