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

// without the skipped segments, or (walked) with those between others: kernels that walk the token axis pass over them
std::vector<Seg> merged(const k82_segments& s, bool walked = false);
// tables of at most kSegs segments with `tile` tokens per tile, which start with their segment or (grid) at multiples of `tile`
std::vector<SegTable> tables(const std::vector<Seg>& segs, int tile, bool grid = false);

// The token sums of the backward passes: the pieces of one index lie side by side (a run), and a run is cut into chunks
// of at most `rows` tokens, whatever the pieces they come from.  One workgroup sums a chunk, a second launch adds the
// chunks of an index in order: no atomics, the same bits every time.  chunk0 numbers the chunks over all tables.
struct RunTable {
    int pieces, runs, rows;
    int start[kSegs], cum[kSegs + 1];          // piece i: tokens [start[i], + cum[i+1] - cum[i]), cum counts over the table
    int index[kSegs], run_cum[kSegs + 1], chunk0[kSegs + 1];
};
// chunks [first[i], first[i+1]) belong to index base + i
struct ReduceTable {
    int base, n;
    int first[kSegs + 1];
};
struct RunPlan {
    std::vector<RunTable> tables;
    std::vector<ReduceTable> reduce;
    int chunks = 0;
};
RunPlan runs(const k82_segments& s, int indices, int rows);
inline int64_t covered(const k82_segments& s) { return s.n ? s.off[s.n] - s.off[0] : 0; }
// at least the chunks that runs() makes
inline int64_t most_chunks(const k82_segments& s, int indices, int rows) {
    const int64_t n = s.n, ends = (n < indices ? n : indices) + n / kSegs + 1;
    return (covered(s) + rows - 1) / rows + ends;
}

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

#define OP_TRY(...)                            \
    do {                                       \
        const hipError_t e_ = (__VA_ARGS__);   \
        if (e_ != hipSuccess) return e_;       \
    } while (0)


typedef uint16_t bf16_t;
typedef uint32_t raw4 __attribute__((ext_vector_type(4)));
// 16 bytes at any address of the element's own alignment: one global_load_dwordx4 / store (the target reads unaligned)
typedef raw4 raw4_any __attribute__((aligned(2)));
typedef raw4 raw4_f __attribute__((aligned(4)));

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {      // round to nearest even, v_cvt_pk_bf16_f32
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    const pair p = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ bf16_t bf16_of(float f) { return (bf16_t)bf16_pair(f, 0.f); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(bf16_t* p, float v) { *p = bf16_of(v); }

// N elements = 16 bytes
template <class T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(raw4 r, float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(r[j]);
    }
    static __device__ __forceinline__ raw4 pack(const float* v) {
        raw4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = __float_as_uint(v[j]);
        return r;
    }
};
template <> struct Vec<bf16_t> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(raw4 r, float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(r[j] << 16); v[2 * j + 1] = __uint_as_float(r[j] & 0xffff0000u); }
    }
    static __device__ __forceinline__ raw4 pack(const float* v) {
        raw4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = bf16_pair(v[2 * j], v[2 * j + 1]);
        return r;
    }
};
// elements [0, n) of the 16 bytes at p, zeros behind them; nothing behind them is read
template <class T> __device__ __forceinline__ raw4 load_part(const T* p, int n) {
    constexpr int N = Vec<T>::N;
    if (n >= N) return *(const raw4_any*)p;
    raw4 r = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (j < n) {
            if constexpr (N == 4) r[j] = __float_as_uint(p[j]);
            else r[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
        }
    return r;
}
template <class T> __device__ __forceinline__ void store_part(T* p, const float* v, int n) {
    constexpr int N = Vec<T>::N;
    if (n >= N) { *(raw4_any*)p = Vec<T>::pack(v); return; }
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (j < n) put(p + j, v[j]);
}

__device__ __forceinline__ float op_gelu_new(float x) {     // the formula of the conv epilogue (conv_mfma_kernel.h), same operations
    const float k = 0.7978845608028654f;
    return 0.5f * x * (1.0f + tanhf(k * (x + 0.044715f * x * x * x)));
}
// how many of v[1 .. kSegs] are <= x (two per lane, one ballot each): the piece a position falls into
__device__ __forceinline__ int place(const int* v, int x) {
    const int lane = threadIdx.x & 63;
    return __popcll(__ballot(v[1 + lane] <= x)) + __popcll(__ballot(v[65 + lane] <= x));
}
__device__ __forceinline__ int seg_of(const op::SegTable& s, int tile) { return place(s.tile0, tile); }
template <int CTRL> __device__ __forceinline__ float lane_move(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// sum over the wave, every lane active: quads, halves and rows of 16 by data-parallel moves, then the four rows
__device__ __forceinline__ float wave_total(float v) {
    v += lane_move<0xb1>(v);                   // lane ^ 1
    v += lane_move<0x4e>(v);                   // lane ^ 2
    v += lane_move<0x141>(v);                  // mirrored in 8
    v += lane_move<0x140>(v);                  // mirrored in 16
    const int i = __float_as_int(v);
    return (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16))) +
           (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
}
