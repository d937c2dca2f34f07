// Operators on caller-owned device tensors: low-rank adapters of many requests beside a shared projection (lora.hip) and
// layer norm with a gain / offset per request (norm.hip), forward and backward.  Host side: argument checks and workspace
// sizes (no GPU needed) and the launches; engine.hip wraps them in the C-ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/k82.h"

namespace op {

// A launch carries its segment table in the kernel arguments (no upload, nothing to keep alive, capturable): at most
// kSegs pieces, longer lists are cut into several launches.  Empty segments are dropped, neighbours of one index merged.
constexpr int kSegs = 128;
struct SegTable {
    int n;
    int start[kSegs], len[kSegs], index[kSegs];
    int tile0[kSegs + 1];                      // first tile of segment i; tile0[i] = tile0[n] for i >= n
};
struct Seg { int start, len, index; };

std::vector<Seg> merged(const k82_segments& s);
// tables of at most kSegs segments with `tile` tokens per tile
std::vector<SegTable> tables(const std::vector<Seg>& segs, int tile);

std::string check(const k82_lora* p, const k82_segments* s);
std::string check(const k82_lora_grad* p, const k82_segments* s);
std::string check(const k82_layernorm* p, const k82_segments* s);
std::string check(const k82_layernorm_grad* p, const k82_segments* s);
int64_t workspace(const k82_lora_grad& p, const k82_segments& s);
int64_t workspace(const k82_layernorm_grad& p, const k82_segments& s);
hipError_t launch(const k82_lora& p, const k82_segments& s, hipStream_t st);
hipError_t launch(const k82_lora_grad& p, const k82_segments& s, void* ws, hipStream_t st);
hipError_t launch(const k82_layernorm& p, const k82_segments& s, hipStream_t st);
hipError_t launch(const k82_layernorm_grad& p, const k82_segments& s, void* ws, hipStream_t st);

template <class... P, class... A> hipError_t run(void (*k)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t st, A... a) {
    std::tuple<P...> v{static_cast<P>(a)...};
    void* args[sizeof...(P)];
    std::apply([&](auto&... x) { int i = 0; ((args[i++] = (void*)&x), ...); }, v);
    return hipLaunchKernel((const void*)k, grid, block, args, lds, st);
}

}  // namespace op

#define OP_TRY(x)                              \
    do {                                       \
        const hipError_t e_ = (x);             \
        if (e_ != hipSuccess) return e_;       \
    } while (0)


typedef uint16_t bf16_t;
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ bf16_t bf16_of(float f) {        // round to nearest even, NaN stays NaN
    const uint32_t u = __float_as_uint(f);
    return (u & 0x7fffffffu) > 0x7f800000u ? (bf16_t)((u >> 16) | 0x40) : (bf16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(bf16_t* p, float v) { *p = bf16_of(v); }
__device__ __forceinline__ float op_gelu_new(float x) {     // the formula of the conv epilogue (conv_mfma_kernel.h), same operations
    const float k = 0.7978845608028654f;
    return 0.5f * x * (1.0f + tanhf(k * (x + 0.044715f * x * x * x)));
}
// segment of tile `tile`: the number of tile0 entries after the first that are <= tile (two per lane, one ballot each)
__device__ __forceinline__ int seg_of(const op::SegTable& s, int tile) {
    const int lane = threadIdx.x & 63;
    const unsigned long long a = __ballot(s.tile0[1 + lane] <= tile), b = __ballot(s.tile0[65 + lane] <= tile);
    return __popcll(a) + __popcll(b);
}
__device__ __forceinline__ float wave_total(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
