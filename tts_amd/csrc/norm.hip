// Layer norm with a gain / offset per segment: z = x + res, y = (z - mean) rstd gain_k + offset_k, and its gradients.
#include "operators.h"

namespace {
using op::SegTable;

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

// Simple form: one workgroup per token, the row read three times.
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

// The weight's gradient first (dx may overwrite an input): one thread per channel and gain, the tokens in order, 64-bit sums
template <class T> __global__ __launch_bounds__(256) void norm_grad_weight_kernel(SegTable sg, k82_layernorm_grad p, int first) {
    const int c = blockIdx.x * 256 + threadIdx.x, k = blockIdx.y;
    if (c >= p.c) return;
    float *dg = p.dgain + (int64_t)k * p.c + c, *db = p.doffset + (int64_t)k * p.c + c;
    double a = first ? 0.0 : (double)*dg, b = first ? 0.0 : (double)*db;
    for (int s = 0; s < sg.n; ++s) {
        if (sg.index[s] != k) continue;
        for (int64_t t = sg.start[s]; t < (int64_t)sg.start[s] + sg.len[s]; ++t) {
            float z = to_f(((const T*)p.x)[t * p.ldx + c]);
            if (p.res) z += to_f(((const T*)p.res)[t * p.ldres + c]);
            const float dy = to_f(((const T*)p.dy)[t * p.lddy + c]);
            a += (double)dy * ((z - p.mean[t]) * p.rstd[t]);
            b += (double)dy;
        }
    }
    *dg = (float)a;
    *db = (float)b;
}
template <class T> __global__ __launch_bounds__(256) void norm_grad_token_kernel(SegTable sg, k82_layernorm_grad p) {
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
    for (int c = threadIdx.x; c < p.c; c += 256) {
        const float xh = (to_f(x[c]) + (res ? to_f(res[c]) : 0.f) - mean) * rstd, u = to_f(dy[c]) * to_f(g[c]);
        put((T*)p.dx + t * p.lddx + c, rstd * (u - v - xh * w));
    }
}

template <class T> hipError_t forward(const k82_layernorm& p, const k82_segments& s, hipStream_t st) {
    const bool cols = p.layout == K82_COLS;
    for (const SegTable& t : op::tables(op::merged(s), 1))
        OP_TRY(op::run(norm_token_kernel<T>, dim3(t.tile0[t.n]), dim3(256), 0, st, t, p, cols ? 1 : p.ldx, cols ? p.ldx : 1,
                       cols ? 1 : p.ldres, cols ? p.ldres : 1, cols ? 1 : p.ldy, cols ? p.ldy : 1));
    return hipSuccess;
}
template <class T> hipError_t backward(const k82_layernorm_grad& p, const k82_segments& s, hipStream_t st) {
    std::vector<SegTable> tabs = op::tables(op::merged(s), 1);
    if (tabs.empty()) { tabs.emplace_back(); tabs[0].n = 0; }
    for (size_t i = 0; i < tabs.size(); ++i)
        OP_TRY(op::run(norm_grad_weight_kernel<T>, dim3((p.c + 255) / 256, p.gains), dim3(256), 0, st, tabs[i], p, i == 0));
    for (const SegTable& t : tabs)
        if (t.n) OP_TRY(op::run(norm_grad_token_kernel<T>, dim3(t.tile0[t.n]), dim3(256), 0, st, t, p));
    return hipSuccess;
}
}  // namespace

namespace op {
int64_t workspace(const k82_layernorm_grad&, const k82_segments&) { return 0; }
hipError_t launch(const k82_layernorm& p, const k82_segments& s, hipStream_t st) {
    return p.dtype == K82_F32 ? forward<float>(p, s, st) : forward<bf16_t>(p, s, st);
}
hipError_t launch(const k82_layernorm_grad& p, const k82_segments& s, void*, hipStream_t st) {
    return p.dtype == K82_F32 ? backward<float>(p, s, st) : backward<bf16_t>(p, s, st);
}
}  // namespace op
