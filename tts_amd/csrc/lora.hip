// Low-rank adapters of many requests beside a shared projection:
//   y_t = act(base_t + s_k B_k (A_k x_t)),  k = index of the token's segment, and the gradients of it.
#include "operators.h"

namespace {
using op::SegTable;

// Simple form: one workgroup per token.  h = A_k x by one wave per factor row, then one thread per output channel.
template <class T>
__global__ __launch_bounds__(256) void lora_token_kernel(SegTable sg, k82_lora p, int64_t xt, int64_t xc, int64_t bt, int64_t bc, int64_t yt, int64_t yc) {
    __shared__ float h[K82_LORA_MAX_RANK];
    const int s = seg_of(sg, blockIdx.x), k = sg.index[s], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = sg.start[s] + ((int)blockIdx.x - sg.tile0[s]);
    const T* x = (const T*)p.x + t * xt;
    if (k >= 0) {
        const T* a = (const T*)p.a + (int64_t)k * p.rank * p.cin;
        for (int r = wave; r < p.rank; r += 4) {
            float v = 0.f;
            for (int c = lane; c < p.cin; c += 64) v = fmaf(to_f(a[(int64_t)r * p.cin + c]), to_f(x[c * xc]), v);
            v = wave_total(v);
            if (lane == 0) h[r] = v;
        }
    } else if (threadIdx.x < K82_LORA_MAX_RANK) h[threadIdx.x] = 0.f;
    __syncthreads();
    if (p.h && threadIdx.x < p.rank) p.h[t * p.rank + threadIdx.x] = h[threadIdx.x];
    const float scale = k >= 0 ? p.scale[k] : 0.f;
    for (int o = threadIdx.x; o < p.cout; o += 256) {
        float v = 0.f;
        if (k >= 0) {
            const T* b = (const T*)p.b + ((int64_t)k * p.cout + o) * p.rank;
            for (int r = 0; r < p.rank; ++r) v = fmaf(to_f(b[r]), h[r], v);
            v *= scale;
        }
        if (p.base) v += to_f(((const T*)p.base)[t * bt + o * bc]);
        if (p.act == K82_ACT_GELU_NEW) v = op_gelu_new(v);
        put((T*)p.y + t * yt + o * yc, v);
    }
}

// g = s_k dy B_k into the workspace, dx = dx_base + g A_k
template <class T> __global__ __launch_bounds__(256) void lora_grad_token_kernel(SegTable sg, k82_lora_grad p, float* g_out) {
    __shared__ float g[K82_LORA_MAX_RANK];
    const int s = seg_of(sg, blockIdx.x), k = sg.index[s], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = sg.start[s] + ((int)blockIdx.x - sg.tile0[s]);
    const T* dy = (const T*)p.dy + t * p.lddy;
    if (k >= 0) {
        const T* b = (const T*)p.b + (int64_t)k * p.cout * p.rank;
        for (int r = wave; r < p.rank; r += 4) {
            float v = 0.f;
            for (int o = lane; o < p.cout; o += 64) v = fmaf(to_f(b[(int64_t)o * p.rank + r]), to_f(dy[o]), v);
            v = wave_total(v);
            if (lane == 0) g_out[t * p.rank + r] = g[r] = v * p.scale[k];
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.cin; c += 256) {
        float v = p.dx_base ? to_f(((const T*)p.dx_base)[t * p.lddx_base + c]) : 0.f;
        if (k >= 0) {
            const T* a = (const T*)p.a + (int64_t)k * p.rank * p.cin + c;
            for (int r = 0; r < p.rank; ++r) v = fmaf(to_f(a[(int64_t)r * p.cin]), g[r], v);
        }
        put((T*)p.dx + t * p.lddx + c, v);
    }
}
// da, db: one thread per element of an adapter's factors, the tokens of its segments in order, sums in 64 bits
template <class T> __global__ __launch_bounds__(256) void lora_grad_weight_kernel(SegTable sg, k82_lora_grad p, const float* g, int first) {
    const int i = blockIdx.x * 256 + threadIdx.x, r = blockIdx.y, k = blockIdx.z;
    if (i >= p.cin + p.cout) return;
    const bool in = i < p.cin;
    float* out = in ? p.da + ((int64_t)k * p.rank + r) * p.cin + i : p.db + ((int64_t)k * p.cout + (i - p.cin)) * p.rank + r;
    double v = first ? 0.0 : (double)*out;
    for (int s = 0; s < sg.n; ++s) {
        if (sg.index[s] != k) continue;
        for (int64_t t = sg.start[s]; t < (int64_t)sg.start[s] + sg.len[s]; ++t)
            v += in ? (double)g[t * p.rank + r] * to_f(((const T*)p.x)[t * p.ldx + i])
                    : (double)(p.scale[k] * p.h[t * p.rank + r]) * to_f(((const T*)p.dy)[t * p.lddy + (i - p.cin)]);
    }
    *out = (float)v;
}

template <class T> hipError_t forward(const k82_lora& p, const k82_segments& s, hipStream_t st) {
    const bool cols = p.layout == K82_COLS;
    for (const SegTable& t : op::tables(op::merged(s), 1))
        OP_TRY(op::run(lora_token_kernel<T>, dim3(t.tile0[t.n]), dim3(256), 0, st, t, p, cols ? 1 : p.ldx, cols ? p.ldx : 1,
                       cols ? 1 : p.ldbase, cols ? p.ldbase : 1, cols ? 1 : p.ldy, cols ? p.ldy : 1));
    return hipSuccess;
}
template <class T> hipError_t backward(const k82_lora_grad& p, const k82_segments& s, void* ws, hipStream_t st) {
    std::vector<SegTable> tabs = op::tables(op::merged(s), 1);
    for (const SegTable& t : tabs)
        OP_TRY(op::run(lora_grad_token_kernel<T>, dim3(t.tile0[t.n]), dim3(256), 0, st, t, p, (float*)ws));
    if (tabs.empty()) { tabs.emplace_back(); tabs[0].n = 0; }
    if (p.adapters > 0)
        for (size_t i = 0; i < tabs.size(); ++i)
            OP_TRY(op::run(lora_grad_weight_kernel<T>, dim3((p.cin + p.cout + 255) / 256, p.rank, p.adapters), dim3(256), 0, st, tabs[i], p,
                           (const float*)ws, i == 0));
    return hipSuccess;
}
}  // namespace

namespace op {
int64_t workspace(const k82_lora_grad& p, const k82_segments&) { return p.tokens * p.rank * 4; }
hipError_t launch(const k82_lora& p, const k82_segments& s, hipStream_t st) {
    return p.dtype == K82_F32 ? forward<float>(p, s, st) : forward<bf16_t>(p, s, st);
}
hipError_t launch(const k82_lora_grad& p, const k82_segments& s, void* ws, hipStream_t st) {
    return p.dtype == K82_F32 ? backward<float>(p, s, ws, st) : backward<bf16_t>(p, s, ws, st);
}
}  // namespace op
