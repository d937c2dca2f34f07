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
// Operands reach the matrix units through LDS: a wave reads 16 rows x 64 bytes with four neighbouring lanes on each row (16
// requests to the cache; a lane a row, as the instruction wants it, would be 64), and takes them from LDS in the instruction's
// order.  The 16-byte places of a row are turned by row / 4, so neither side meets a bank twice.  The region belongs to one
// wave, whose LDS accesses happen in order: no barrier.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// 16 bytes at a uniform base and a lane's own 32-bit offset (one register a lane for an address; rows are at most 2^25 long)
__device__ __forceinline__ raw4 load16(const char* base, uint32_t at) { return *(const raw4_any*)(base + at); }
// The same at a place that may lie in part (EVEN: as a whole) behind the row: n elements from there on are in the row, `back`
// bytes before it there is some.
template <class T, bool EVEN> __device__ __forceinline__ raw4 grab(const char* base, uint32_t at, int n, uint32_t back) {
    if constexpr (EVEN) {
        const raw4 r = load16(base, n > 0 ? at : at - back), zero = {0u, 0u, 0u, 0u};
        return n > 0 ? r : zero;
    } else return n > 0 ? load_part((const T*)(base + at), n) : raw4{0u, 0u, 0u, 0u};
}
// the elements 0, ld, 2 ld ... of p as 16 bytes: n of them at most, zeros behind
template <class T> __device__ __forceinline__ raw4 across(const T* p, int ld, int n) {
    constexpr int N = Vec<T>::N;
    T v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < n ? p[j * (uint32_t)ld] : T(0);
    raw4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (N == 4) r[j] = __float_as_uint(v[j]);
        else r[j] = v[2 * j] | (uint32_t)v[2 * j + 1] << 16;
    }
    return r;
}
__device__ __forceinline__ void put_tile(raw4* tile, raw4 v) {
    const int lane = threadIdx.x & 63;
    tile[(lane & ~3) + ((lane & 3) ^ (lane >> 4))] = v;
}
__device__ __forceinline__ raw4 get_tile(const raw4* tile) {
    const int col = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    return tile[4 * col + (g ^ (col >> 2))];
}

// The factor rank in tiles: RT of 16 rows.  From two on, bf16 pairs them so that a lane's h are 8 consecutive ranks: row m of
// tile 2 j + e is the rank 32 j + 8 (m / 4) + 4 e + m % 4.
template <class T, int RT> __device__ __forceinline__ int rank_of(int tile, int row) {
    if constexpr (Vec<T>::N == 8 && RT > 1) return 32 * (tile >> 1) + 8 * (row >> 2) + 4 * (tile & 1) + (row & 3);
    return 16 * tile + row;
}
// v as far as a finite bf16 goes, and two of them as a part.  What is left behind a part is then a difference of finite numbers
// where v is finite, also next to the largest f32, which alone would round to an infinity; where it is not, the last part is.
__device__ __forceinline__ float in_bf16(float v) { return __builtin_amdgcn_fmed3f(v, -0x1.fep127f, 0x1.fep127f); }
__device__ __forceinline__ uint32_t finite_pair(float a, float b) { return bf16_pair(in_bf16(a), in_bf16(b)); }
// h as the second product's operand, and that product of one row tile of B with one tile of tokens.
// f32: itself.  bf16: in two parts, h = hi + lo to 2^-16 (rounded to one part alone, h would cost half of the result's own
// precision); at one tile both parts share an instruction, with B's four values twice.
template <class T, int RT> struct Second;
template <int RT> struct Second<float, RT> {
    static constexpr int CHUNKS = RT;          // 64-byte chunks of a row of B
    raw4 v[RT];
    __device__ __forceinline__ void set(const f4 (&h)[RT]) {
#pragma unroll
        for (int r = 0; r < RT; ++r) v[r] = __builtin_bit_cast(raw4, h[r]);
    }
    __device__ __forceinline__ f4 times(const raw4 (&b)[CHUNKS], f4 d) const {
#pragma unroll
        for (int r = 0; r < RT; ++r) d = product<float>(b[r], v[r], d);
        return d;
    }
};
template <int RT> struct Second<bf16_t, RT> {
    static constexpr int CHUNKS = (RT + 1) / 2;
    raw4 v[RT];                                // RT = 1: hi | lo; else hi and lo of each pair
    static __device__ __forceinline__ void parts(const f4& h, uint32_t* hi, uint32_t* lo) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            hi[j] = finite_pair(h[2 * j], h[2 * j + 1]);
            lo[j] = bf16_pair(h[2 * j] - __uint_as_float(hi[j] << 16), h[2 * j + 1] - __uint_as_float(hi[j] & 0xffff0000u));
        }
    }
    __device__ __forceinline__ void set(const f4 (&h)[RT]) {
        uint32_t hi[RT][2], lo[RT][2];
#pragma unroll
        for (int r = 0; r < RT; ++r) parts(h[r], hi[r], lo[r]);
        if constexpr (RT == 1) v[0] = raw4{hi[0][0], hi[0][1], lo[0][0], lo[0][1]};
        else
#pragma unroll
            for (int r = 0; r < RT; r += 2) {
                v[r] = raw4{hi[r][0], hi[r][1], hi[r + 1][0], hi[r + 1][1]};
                v[r + 1] = raw4{lo[r][0], lo[r][1], lo[r + 1][0], lo[r + 1][1]};
            }
    }
    __device__ __forceinline__ f4 times(const raw4 (&b)[CHUNKS], f4 d) const {
        if constexpr (RT == 1) return product<bf16_t>(b[0], v[0], d);
#pragma unroll
        for (int r = 0; r < RT; ++r) d = product<bf16_t>(b[r >> 1], v[r], d);
        return d;
    }
};
// a row tile of B from LDS: chunk j as times() takes it
template <class T, int RT> __device__ __forceinline__ raw4 get_factor(const raw4* tile) {
    if constexpr (Vec<T>::N == 8 && RT == 1) {                   // ranks 4 g .. 4 g + 3, twice
        const int col = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
        const raw2 r = ((const raw2*)(tile + 4 * col + ((g >> 1) ^ (col >> 2))))[g & 1];
        return raw4{r[0], r[1], r[0], r[1]};
    } else return get_tile(tile);
}

// two tiles side by side, 128 bytes of each row: the 16 bytes of the row 8 e + lane / 8; tile e as the operand
__device__ __forceinline__ void put_pair(raw4* tiles, int e, raw4 v) {
    const int lane = threadIdx.x & 63;
    tiles[64 * e + (lane & ~7) + ((lane & 7) ^ (lane >> 3))] = v;
}
__device__ __forceinline__ raw4 get_pair(const raw4* tiles, int e) {
    const int col = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    return tiles[8 * col + ((4 * e + g) ^ (col & 7))];
}

// The sum over the waves' parts of k, and what follows from it for every wave: h for the second product, and h itself if kept.
// tok: the token of this lane's column.
template <class T, int NW, int RT, int TT>
__device__ __forceinline__ void join(f4 (*part)[RT * TT][64], f4 (&acc)[RT][TT], Second<T, RT> (&h)[TT], int rank, float scale, float* keep, const int64_t* tok, const bool* in) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < TT; ++t) part[wave][r * TT + t][lane] = acc[r][t];
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        f4 sum[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int i = r * TT + t;
            f4 v = part[0][i][lane];
#pragma unroll 3
            for (int w = 1; w < NW; ++w) v += part[w][i][lane];
            const int r0 = rank_of<T, RT>(r, 4 * g);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r0 + j >= rank) v[j] = 0.f;                  // rows of A behind the rank were read from its last row
            if (keep && wave == i % NW && in[t]) {
                float* q = keep + tok[t] * rank + r0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (r0 + j < rank) q[j] = v[j];
            }
            sum[r] = v * scale;
        }
        h[t].set(sum);
    }
    __syncthreads();                                             // the parts' memory is used again
}

constexpr int most(int a, int b) { return a > b ? a : b; }
constexpr int kPad = 4;                        // floats behind a row of the results' tile: rows start on different banks

// Token rows.  A workgroup takes 16 TT tokens of a segment; its NW waves share the k of the first product (each takes every
// NW-th 128 bytes of a row: whole lines, 8 a load and not 16; 65536 tokens 2048 -> 768 bf16 rank 64 with TT = 2 133 us, with 64 bytes
// 139) and the output channels of the second, 128 bytes of a row a wave at a time.  The results cross LDS once more, so that base and y are read and written in whole lines.
// blockIdx.y splits the output channels where there are few tokens; each part then computes h for itself, from cache.
// EVEN: cin, cout and rank are multiples of a lane's 16 bytes, no place lies in part behind a row.
// A step's registers are loaded again as soon as LDS has its operands; a second step in flight fits only one rank tile (with
// two it spilled: 65536 tokens 768 -> 768 bf16 rank 32 81 us, without 64).
// The call above with TT = 4: 127 us of 473 MB, 3.7 TB/s (a large copy: 4.7).
// (waves_per_eu: without it accumulators are copied through the second register file and a wave less fits a SIMD.)
// ACROSS: a is [adapters][cin][rank] and b [adapters][rank][cout], read element by element (the backward pass of one rank tile).
template <class T, int NW, int RT, int TT, bool EVEN, bool ACROSS = false>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(RT >= 8 ? 1 : RT >= 4 ? 2 : 4))) void lora_rows_kernel(SegTable sg, k82_lora p) {
    constexpr int V = Vec<T>::N, K = 4 * V, K2 = 2 * K, S = sizeof(T), U = RT > 1 ? 1 : 2;          // a step: 128 bytes of a row; U of them in flight
    constexpr int CH = 8 * V, MT = CH / 16, CK = Second<T, RT>::CHUNKS;          // channels, row tiles of B, chunks of a row of B
    constexpr int kTiles = most(2 * (RT + TT), MT * CK), kRow = CH + kPad;
    constexpr int kOwn = most(kTiles * 1024, MT * CK * 1024 + 16 * kRow * 4);    // a wave's own bytes
    __shared__ __align__(16) char lds[most(NW * kOwn, NW * RT * TT * 1024)];
    const int s = seg_of(sg, blockIdx.x), k = sg.index[s];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    if (k < 0 && p.act == K82_ACT_NONE && p.base == p.y && !p.h) return;
    raw4* own = (raw4*)(lds + wave * kOwn);
    float* result = (float*)(own + MT * CK * 64);
    const int row0 = ((int)blockIdx.x - sg.tile0[s]) * 16 * TT, last = sg.len[s] - 1 - row0;
    const int64_t t0 = sg.start[s] + row0;
    // Second product: this lane's 16 bytes of the tokens (lane / 8) + 8 i
    const int blocks = (p.cout + CH - 1) / CH, stride = NW * gridDim.y, c8 = V * (lane & 7), c4 = V * (lane & 3);
    const char* basep = (const char*)p.base + t0 * p.ldbase * S;
    char* yp = (char*)p.y + t0 * p.ldy * S;
    const char* bp = (const char*)p.b + (int64_t)max(k, 0) * p.cout * p.rank * S;
    int blk = (int)blockIdx.y * NW + wave;
    raw4 base[2 * TT], fac[MT * CK];
    auto fetch = [&](int blk) {
        const int n = p.cout - blk * CH;
        if (p.base) {
#pragma unroll
            for (int i = 0; i < 2 * TT; ++i)
                base[i] = grab<T, EVEN>(basep + (int64_t)blk * CH * S, (min(8 * i + (lane >> 3), last) * (uint32_t)p.ldbase + c8) * S, n - c8, c8 * S);
        }
        if (k >= 0) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int row = min(16 * m + (lane >> 2), n - 1);
                const uint32_t at = (row * (uint32_t)p.rank + c4) * S;
#pragma unroll
                for (int c = 0; c < CK; ++c)
                    if constexpr (ACROSS) fac[m * CK + c] = across((const T*)(bp + (int64_t)blk * CH * S) + row + (uint32_t)(c * K + c4) * p.cout, p.cout, p.rank - c * K - c4);
                    else fac[m * CK + c] = grab<T, EVEN>(bp + (int64_t)blk * CH * p.rank * S, at + c * K * S, p.rank - c * K - c4, (c * K + c4) * S);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < 2 * TT; ++i) base[i] = raw4{0u, 0u, 0u, 0u};
    if (blk < blocks) fetch(blk);
    Second<T, RT> h[TT];
    if (k >= 0) {
        f4 acc[RT][TT];
        const char *ap = (const char*)p.a + (int64_t)k * p.rank * p.cin * S, *xp = (const char*)p.x + t0 * p.ldx * S;
        uint32_t ao[RT][2], xo[TT][2];                           // this lane's 16 bytes of the rows (lane / 8) and + 8 of a tile
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = 8 * e + (lane >> 3);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const uint32_t k = min(rank_of<T, RT>(r, row), p.rank - 1);
                ao[r][e] = (ACROSS ? c8 * (uint32_t)p.rank + k : k * (uint32_t)p.cin + c8) * S;
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) xo[t][e] = (min(16 * t + row, last) * (uint32_t)p.ldx + c8) * S;
        }
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[r][t] = f4{0.f, 0.f, 0.f, 0.f};
        raw4 fa[U][RT][2], fx[U][TT][2];
        const int full = p.cin / K2;
        auto load = [&](int u, int i) {
            const int at = i * K2 * S;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int t = 0; t < TT; ++t) fx[u][t][e] = load16(xp + at, xo[t][e]);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    if constexpr (ACROSS) fa[u][r][e] = across((const T*)(ap + (int64_t)at * p.rank + ao[r][e]), p.rank, V);
                    else fa[u][r][e] = load16(ap + at, ao[r][e]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);                   // (the compiler would gather the loads of several steps)
        };
        // step u of the ring, whose place then takes step `next` (sure: there is one)
        auto multiply = [&](int u, int next, auto sure) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int t = 0; t < TT; ++t) put_pair(own + t * 128, e, fx[u][t][e]);
#pragma unroll
                for (int r = 0; r < RT; ++r) put_pair(own + (TT + r) * 128, e, fa[u][r][e]);
            }
            if (decltype(sure)::value || next < full) load(u, next);
            wave_fence();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                raw4 ta[RT], tx[TT];
#pragma unroll
                for (int t = 0; t < TT; ++t) tx[t] = get_pair(own + t * 128, e);
#pragma unroll
                for (int r = 0; r < RT; ++r) ta[r] = get_pair(own + (TT + r) * 128, e);
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int t = 0; t < TT; ++t) acc[r][t] = product<T>(ta[r], tx[t], acc[r][t]);
            }
            wave_fence();
        };
        int i = wave;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * NW < full) load(u, i + u * NW);
        for (; i + (2 * U - 1) * NW < full; i += U * NW) {
#pragma unroll
            for (int u = 0; u < U; ++u) multiply(u, i + (U + u) * NW, std::true_type());
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i < full) { multiply(u, i + U * NW, std::false_type()); i += NW; }
#pragma unroll
        for (int u = 0; u < U - 1; ++u)
            if (i < full) { multiply(u, full, std::false_type()); i += NW; }
        if (i == full && p.cin % K2) {                           // one wave: the end of the row, zeros behind it
            const int at = full * K2 * S, n = p.cin - full * K2 - c8;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int t = 0; t < TT; ++t) fx[0][t][e] = grab<T, EVEN>(xp + at, xo[t][e], n, c8 * S);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    if constexpr (ACROSS) fa[0][r][e] = across((const T*)(ap + (int64_t)at * p.rank + ao[r][e]), p.rank, n);
                    else fa[0][r][e] = grab<T, EVEN>(ap + at, ao[r][e], n, c8 * S);
                }
            }
            multiply(0, full, std::false_type());
        }
        int64_t tok[TT];
        bool in[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) { tok[t] = t0 + 16 * t + col; in[t] = 16 * t + col <= last; }
        join<T, NW, RT, TT>((f4(*)[RT * TT][64])lds, acc, h, p.rank, p.scale[k], blockIdx.y == 0 ? p.h : nullptr, tok, in);
    } else if (p.h && blockIdx.y == 0) {
        const int n = min(16 * TT, last + 1) * p.rank;
        for (int i = threadIdx.x; i < n; i += 64 * NW) p.h[t0 * p.rank + i] = 0.f;
    }
    for (; blk < blocks; blk += stride) {
        raw4 now[2 * TT];
#pragma unroll
        for (int i = 0; i < 2 * TT; ++i) now[i] = base[i];
        if (k >= 0) {
#pragma unroll
            for (int i = 0; i < MT * CK; ++i) put_tile(own + i * 64, fac[i]);
        }
        if (blk + stride < blocks) fetch(blk + stride);          // the next block is on its way while this one is multiplied
        const int n = p.cout - blk * CH - c8;
        char* yb = yp + (int64_t)blk * CH * S;
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            if (k >= 0) {
                wave_fence();
#pragma unroll
                for (int m = 0; m < MT; ++m) {                   // (B's tiles are read for each t: registers for them would cost a wave)
                    raw4 tile[CK];
#pragma unroll
                    for (int c = 0; c < CK; ++c) tile[c] = get_factor<T, RT>(own + (m * CK + c) * 64);
                    *(f4*)(result + col * kRow + 16 * m + 4 * g) = h[t].times(tile, f4{0.f, 0.f, 0.f, 0.f});
                }
                wave_fence();
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float f[V];
                Vec<T>::unpack(now[2 * t + i], f);
                if (k >= 0) {
#pragma unroll
                    for (int j = 0; j < V; j += 4) {
                        const f4 d = *(const f4*)(result + (8 * i + (lane >> 3)) * kRow + c8 + j);
                        f[j] += d[0]; f[j + 1] += d[1]; f[j + 2] += d[2]; f[j + 3] += d[3];
                    }
                }
                if (p.act == K82_ACT_GELU_NEW)
#pragma unroll
                    for (int j = 0; j < V; ++j) f[j] = op_gelu_new(f[j]);
                const int row = 16 * t + 8 * i + (lane >> 3);
                if (row <= last && n > 0) {
                    T* q = (T*)(yb + (row * (uint32_t)p.ldy + c8) * S);
                    if constexpr (EVEN) *(raw4_any*)q = Vec<T>::pack(f);
                    else store_part(q, f, n);
                }
            }
            wave_fence();
        }
    }
}

// Channel-first: the same products, TT consecutive tokens a lane (tile t of a lane's tokens is TT col + t), 16 TT tokens a
// workgroup, on the token grid of the tensor.  A tile that holds several segments has a workgroup for each (one that
// walked them took twice as long as the others, and the launch as long as it: 16411 x 768 in 64 sentences 48 us, now 42);
// what is loaded of the others' tokens stays in its own columns and is not stored.
// The last tile reads at the tensor's end (t = its last pair, or token) and takes what is left: `second` where that pair is one
// token ahead of the lane's.  at: bytes of the row
template <int TT> __device__ __forceinline__ void load_tokens(float (&v)[TT], const char* base, uint32_t at, bool second) {
    if constexpr (TT == 2) {
        const f2_any r = *(const f2_any*)(base + at);
        v[0] = second ? r[1] : r[0];
        v[1] = r[1];
    } else v[0] = *(const float*)(base + at);
}
// (waves_per_eu as above: 65536 x 768 rank 32 192 us, with it 165.)
template <int NW, int RT, int TT, bool EVEN>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(RT >= 8 ? 2 : RT >= 4 ? 3 : 4))) void lora_cols_kernel(SegTable sg, k82_lora p) {
    constexpr int U = 2;
    __shared__ __align__(16) char lds[most(NW * RT * 1024, NW * RT * TT * 1024)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    raw4* own = (raw4*)lds + wave * RT * 64;
    const int s = seg_of(sg, blockIdx.x), k = sg.index[s], lo = sg.start[s], hi = lo + sg.len[s];
    if (k < 0 && p.act == K82_ACT_NONE && p.base == p.y && !p.h) return;
    const int tokens = (int)p.tokens, c4 = 4 * (lane & 3);
    const int tile = lo / (16 * TT) * (16 * TT) + ((int)blockIdx.x - sg.tile0[s]) * 16 * TT, t0 = tile + TT * col;
    const uint32_t tb = 4 * min(t0, tokens - TT);
    const bool second = t0 == tokens - 1;
    // the lane's four channels (4 g + i) of 16 from base on, n of them there; behind those any that is (EVEN: four at a time, so
    // that one register holds the lane's offset)
    auto load_rows = [&](float (&v)[4][TT], const char* base, int64_t ld, int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (EVEN) load_tokens<TT>(v[i], base + i * ld * 4, min(4 * g, n - 4) * (uint32_t)ld * 4 + tb, second);
            else load_tokens<TT>(v[i], base, min(4 * g + i, n - 1) * (uint32_t)ld * 4 + tb, second);
        }
    };
    const int blocks = (p.cout + 15) / 16, stride = NW * gridDim.y;
    int blk = (int)blockIdx.y * NW + wave;
    float base[4][TT];
    raw4 fac[RT];
    const char* bp = (const char*)p.b + (int64_t)max(k, 0) * p.cout * p.rank * 4;
    auto fetch = [&](int blk) {
        const int n = p.cout - 16 * blk;
        if (p.base) {
            const char* q = (const char*)p.base + (int64_t)16 * blk * p.ldbase * 4;
            load_rows(base, q, p.ldbase, n);
        }
        if (k >= 0) {
            const uint32_t at = (min(lane >> 2, n - 1) * (uint32_t)p.rank + c4) * 4;
#pragma unroll
            for (int r = 0; r < RT; ++r) fac[r] = grab<float, EVEN>(bp + (int64_t)16 * blk * p.rank * 4, at + 64 * r, p.rank - 16 * r - c4, (16 * r + c4) * 4);
        }
    };
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < TT; ++t) base[i][t] = 0.f;
    if (blk < blocks) fetch(blk);
    Second<float, RT> h[TT];
    if (k >= 0) {
        f4 acc[RT][TT];
        uint32_t ao[RT];
        const char* ap = (const char*)p.a + (int64_t)k * p.rank * p.cin * 4;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            ao[r] = (min(16 * r + (lane >> 2), p.rank - 1) * (uint32_t)p.cin + c4) * 4;
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[r][t] = f4{0.f, 0.f, 0.f, 0.f};
        }
        auto multiply = [&](const raw4 (&fa)[RT], const float (&fx)[4][TT]) {
#pragma unroll
            for (int r = 0; r < RT; ++r) put_tile(own + r * 64, fa[r]);
            wave_fence();
            raw4 ta[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) ta[r] = get_tile(own + r * 64);
            wave_fence();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int t = 0; t < TT; ++t) acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ta[r][i]), fx[i][t], acc[r][t], 0, 0, 0);
        };
        auto steps = [&](int i0, auto n) {                   // 16 channels a step: 4 g + i in instruction i
            constexpr int n_ = decltype(n)::value;
            float fx[n_][4][TT];
            raw4 fa[n_][RT];
#pragma unroll
            for (int u = 0; u < n_; ++u) {
                const int c0 = 16 * (i0 + u * NW);
                const char* q = (const char*)p.x + (int64_t)c0 * p.ldx * 4;
#pragma unroll
                for (int i = 0; i < 4; ++i) load_tokens<TT>(fx[u][i], q + (int64_t)i * p.ldx * 4, 4 * g * (uint32_t)p.ldx * 4 + tb, second);
#pragma unroll
                for (int r = 0; r < RT; ++r) fa[u][r] = load16(ap + 4 * c0, ao[r]);
            }
#pragma unroll
            for (int u = 0; u < n_; ++u) multiply(fa[u], fx[u]);
        };
        const int full = p.cin / 16;
        int i = wave;
        for (; i + (U - 1) * NW < full; i += U * NW) steps(i, std::integral_constant<int, U>());
        if (i < full) { steps(i, std::integral_constant<int, 1>()); i += NW; }
        if (i == full && p.cin % 16) {                       // one wave: the last channels, zeros behind them
            const int c0 = 16 * full, n = p.cin - c0;
            const char* q = (const char*)p.x + (int64_t)c0 * p.ldx * 4;
            raw4 fa[RT];
            float fx[4][TT];
#pragma unroll
            for (int r = 0; r < RT; ++r) fa[r] = grab<float, EVEN>(ap + 4 * c0, ao[r], n - c4, 4 * c4);
            load_rows(fx, q, p.ldx, n);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < TT; ++t) fx[i][t] = 4 * g + i < n ? fx[i][t] : 0.f;
            multiply(fa, fx);
        }
        int64_t tok[TT];
        bool in[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) { tok[t] = t0 + t; in[t] = t0 + t >= lo && t0 + t < hi; }
        join<float, NW, RT, TT>((f4(*)[RT * TT][64])lds, acc, h, p.rank, p.scale[k], blockIdx.y == 0 ? p.h : nullptr, tok, in);
    } else if (p.h && blockIdx.y == 0) {
        const int from = max(tile, lo), n = (min(tile + 16 * TT, hi) - from) * p.rank;
        for (int i = threadIdx.x; i < n; i += 64 * NW) p.h[(int64_t)from * p.rank + i] = 0.f;
    }
    for (; blk < blocks; blk += stride) {
        f4 d[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) d[t] = f4{base[0][t], base[1][t], base[2][t], base[3][t]};
        raw4 fb[RT];
        if (k >= 0) {
#pragma unroll
            for (int r = 0; r < RT; ++r) put_tile(own + r * 64, fac[r]);
            wave_fence();
#pragma unroll
            for (int r = 0; r < RT; ++r) fb[r] = get_tile(own + r * 64);
            wave_fence();
        }
        if (blk + stride < blocks) fetch(blk + stride);      // the next block is on its way while this one is multiplied
        if (k >= 0)
#pragma unroll
            for (int t = 0; t < TT; ++t) d[t] = h[t].times(fb, d[t]);
        char* yb = (char*)p.y + (int64_t)16 * blk * p.ldy * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 4 * g + i;
            float v[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) v[t] = p.act == K82_ACT_GELU_NEW ? op_gelu_new(d[t][i]) : d[t][i];
            if (16 * blk + c >= p.cout) continue;
            float* q = (float*)(yb + (int64_t)i * p.ldy * 4 + (4 * g * (uint32_t)p.ldy + t0) * 4);
            if (t0 >= lo && t0 + TT <= hi) {
                if constexpr (TT == 2) *(f2_any*)q = f2_any{v[0], v[1]};
                else q[0] = v[0];
            } else
#pragma unroll
                for (int t = 0; t < TT; ++t)
                    if (t0 + t >= lo && t0 + t < hi) q[t] = v[t];
        }
    }
}

constexpr int kWaves = 4;                      // of the weight's gradient

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
        hi[j] = finite_pair(a, b);
        a -= __uint_as_float(hi[j] << 16);
        b -= __uint_as_float(hi[j] & 0xffff0000u);
        mid[j] = finite_pair(a, b);
        lo[j] = bf16_pair(a - __uint_as_float(mid[j] << 16), b - __uint_as_float(mid[j] & 0xffff0000u));
    }
}
// Sums over tokens: part[chunk][r][cin + cout] = s_k sum_t v_t[r] z_t[c] with (v, z) = (g / s_k, x) for the first cin channels
// and (h, dy) behind them.  A wave owns 128 channels of one of the two for all the tokens of a chunk.  The token axis is the
// k of the product: f32 takes it as it lies (4 tokens an instruction), bf16 through the transpose in registers.
// More than 32 ranks are shares of neighbouring workgroups (their sums would leave one wave a SIMD): the channels come from the
// shared cache again, 65536 tokens 768 / 2048 rank 64 130 us, with the shares one after the other 173.
// Two steps in flight where the registers of two waves a SIMD hold them (D): the backward pass of 65536 tokens 768 / 2048 rank 8
// bf16 198 -> 184 us; f32 gains nothing from it (32768 tokens 768 / 768 rank 8 115 us either way).
template <class T, int RT, bool EVEN>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2))) void lora_weight_kernel(RunTable rt, k82_lora_grad p, const float* gs, float* part) {
    constexpr int V = Vec<T>::N, M = 8, S = sizeof(T), D = RT == 1 ? 2 : 1;          // M: 16 x 16 tiles along the channels
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int chunk = rt.chunk0[0] + (int)blockIdx.y, run = place(rt.chunk0, chunk);
    const int u0 = rt.run_cum[run] + (chunk - rt.chunk0[run]) * rt.rows, u1 = min(u0 + rt.rows, rt.run_cum[run + 1]);
    // waves of a workgroup: slices of 128 channels; from two rank shares on, two slices by two shares
    const int shares = (p.rank + 31) / 32, pair = shares > 1 ? 2 : 1, groups = (shares + pair - 1) / pair, per = kWaves / pair;
    const int share = (int)blockIdx.x % groups * pair + wave / per, r0 = 32 * share;
    int slice = (int)blockIdx.x / groups * per + wave % per;
    const int nx = (p.cin + 127) / 128, ny = (p.cout + 127) / 128;
    if (slice >= nx + ny || share >= shares) return;
    const bool of_x = slice < nx;
    if (!of_x) slice -= nx;
    const char* z = (const char*)(of_x ? p.x : p.dy);
    const int64_t ld = of_x ? p.ldx : p.lddy;
    const int width = of_x ? p.cin : p.cout, c0 = 128 * slice;
    const float* v = of_x ? gs : p.h;
    f4 acc[M][RT];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[m][r] = f4{0.f, 0.f, 0.f, 0.f};
    // 16 bytes of channel c on at a row (uniform base, the lane's row and channel in `at`); behind the row's end (EVEN: whole
    // places) anything that is there, it is not stored
    auto take = [&](const char* base, uint32_t at, int c) -> raw4 {
        if constexpr (EVEN) return load16(base, at + min(c, width - V) * S);
        else return c < width ? load_part((const T*)(base + at) + c, width - c) : raw4{0u, 0u, 0u, 0u};
    };
    uint32_t rank_at[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) rank_at[r] = min(r0 + 16 * r + col, p.rank - 1);
    // the steps of N tokens of a piece: D of them in flight, each place loaded again as soon as its step is in the operands
    auto ring = [&](auto size, int n, auto& load, auto& use) {
        constexpr int N = decltype(size)::value;
        int i = 0;
#pragma unroll
        for (int b = 0; b < D; ++b)
            if (N * (b + 1) <= n) load(b, N * b, std::true_type());
        for (; i + 2 * D * N <= n; i += D * N)
#pragma unroll
            for (int b = 0; b < D; ++b) use(b, i + (D + b) * N, std::true_type());
#pragma unroll
        for (int b = 0; b < 2 * D - 1; ++b)
            if (i + N <= n) { use(b % D, i + D * N, std::false_type()); i += N; }
        if (i < n) { load(0, i, std::false_type()); use(0, n, std::false_type()); }
    };
    int piece = place(rt.cum, u0);
    for (int u = u0; u < u1; ++piece) {                          // the pieces of a chunk, each a run of neighbouring tokens
        const int stop = min(u1, rt.cum[piece + 1]);
        const int64_t t0 = rt.start[piece] + (u - rt.cum[piece]);
        const int n = stop - u;
        u = stop;
        const char* zp = z + t0 * ld * S;
        const float* vp = v + t0 * p.rank;
        if constexpr (V == 8) {
            raw4 raw[D][8];
            float w[D][RT][8];
            auto load = [&](int b, int i, auto whole) {          // 32 tokens, 8 g + j in a lane; not whole: zeros behind the n-th
                constexpr bool WHOLE = decltype(whole)::value;
                const raw4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int t = i + 8 * g + j;
                    const int at = WHOLE ? i + j : min(i + j, n - 1);
                    const uint32_t row = WHOLE ? 8 * g : max(min(8 * g, n - 1 - at), 0);
                    raw[b][j] = take(zp + (int64_t)at * ld * S, row * (uint32_t)ld * S, c0 + 8 * col);
#pragma unroll
                    for (int r = 0; r < RT; ++r) w[b][r][j] = *(const float*)((const char*)(vp + (int64_t)at * p.rank) + 4 * (row * p.rank + rank_at[r]));
                    if constexpr (!WHOLE) {
                        raw[b][j] = t < n ? raw[b][j] : zero;
#pragma unroll
                        for (int r = 0; r < RT; ++r) w[b][r][j] = t < n ? w[b][r][j] : 0.f;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            auto use = [&](int b, int next, auto sure) {
                raw4 zt[8], w3[RT][3];
                transpose8(raw[b], zt);
#pragma unroll
                for (int r = 0; r < RT; ++r) split3(w[b][r], w3[r][0], w3[r][1], w3[r][2]);
                if (decltype(sure)::value || next + 32 <= n) load(b, next, std::true_type());
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int m = 0; m < 8; ++m)
#pragma unroll
                        for (int q = 2; q >= 0; --q) acc[m][r] = product<T>(zt[m], w3[r][q], acc[m][r]);
            };
            ring(std::integral_constant<int, 32>(), n, load, use);
        } else {
            raw4 raw[D][4][2];
            float w[D][RT][4];
            auto load = [&](int b, int i, auto whole) {          // 16 tokens, 4 j + g in instruction j
                constexpr bool WHOLE = decltype(whole)::value;
                const raw4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int t = i + 4 * j + g, at = WHOLE ? i + 4 * j : min(i + 4 * j, n - 1);
                    const uint32_t row = WHOLE ? g : max(min(g, n - 1 - at), 0);
#pragma unroll
                    for (int m = 0; m < 2; ++m) raw[b][j][m] = take(zp + (int64_t)at * ld * S, row * (uint32_t)ld * S, c0 + 64 * m + 4 * col);
#pragma unroll
                    for (int r = 0; r < RT; ++r) w[b][r][j] = *(const float*)((const char*)(vp + (int64_t)at * p.rank) + 4 * (row * p.rank + rank_at[r]));
                    if constexpr (!WHOLE) {
#pragma unroll
                        for (int m = 0; m < 2; ++m) raw[b][j][m] = t < n ? raw[b][j][m] : zero;
#pragma unroll
                        for (int r = 0; r < RT; ++r) w[b][r][j] = t < n ? w[b][r][j] : 0.f;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            auto use = [&](int b, int next, auto sure) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int m = 0; m < 8; ++m)
                            acc[m][r] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(raw[b][j][m >> 2][m & 3]), w[b][r][j], acc[m][r], 0, 0, 0);
                if (decltype(sure)::value || next + 16 <= n) load(b, next, std::true_type());
            };
            ring(std::integral_constant<int, 16>(), n, load, use);
        }
    }
    // row 4 g + i of tile m is the channel 8 (4 g + i) + m (bf16) or 64 (m / 4) + 4 (4 g + i) + m % 4 (f32)
    const float scale = p.scale[rt.index[run]];
    float* out = part + (int64_t)chunk * p.rank * (p.cin + p.cout) + (of_x ? 0 : p.cin);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        if (r0 + 16 * r + col >= p.rank) continue;
        float* q = out + (int64_t)(r0 + 16 * r + col) * (p.cin + p.cout);
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
// da, db: the chunks of an adapter, 64 channels x 16 ranks a workgroup.  Four shares of four waves take every fourth chunk in
// order, and their sums join in order (4096 tokens of one adapter, 768 / 768 bf16 rank 8, 85 chunks: the backward pass 48 us
// with one share, 29 with four).  db's ranks leave side by side.
__global__ __launch_bounds__(1024) void lora_reduce_kernel(ReduceTable rt, int cin, int cout, int rank, const float* part, float* da, float* db) {
    __shared__ float tile[4][64][17];
    const int nx = (cin + 63) / 64, k = blockIdx.z, r0 = 16 * blockIdx.y;
    const bool of_x = (int)blockIdx.x < nx;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = wave & 3, share = wave >> 2;
    const int width = of_x ? cin : cout, c0 = 64 * ((int)blockIdx.x - (of_x ? 0 : nx)), c = c0 + lane;
    const int64_t step = (int64_t)rank * (cin + cout);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < width) {
        const float* q = part + (int64_t)(rt.first[k] + share) * step + (of_x ? 0 : cin) + c;
        int64_t row[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) row[j] = (int64_t)min(r0 + group + 4 * j, rank - 1) * (cin + cout);
        int n = (rt.first[k + 1] - rt.first[k] - share + 3) / 4;
        for (; n >= 2; n -= 2, q += 8 * step) {                  // (eight loads at once, added in order)
            float v[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = q[4 * i * step + row[j]];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += v[i][j];
        }
        if (n > 0)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += q[row[j]];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) tile[share][lane][group + 4 * j] = s[j];
    __syncthreads();
    const int r = of_x ? wave : threadIdx.x & 15, i = of_x ? lane : threadIdx.x >> 4;
    if (c0 + i >= width || r0 + r >= rank) return;
    const float sum = ((tile[0][i][r] + tile[1][i][r]) + tile[2][i][r]) + tile[3][i][r];
    if (of_x) da[((int64_t)(rt.base + k) * rank + r0 + r) * cin + c0 + i] = sum;
    else db[((int64_t)(rt.base + k) * cout + c0 + i) * rank + r0 + r] = sum;
}

template <class F> hipError_t by_rank(int rank, F&& f) {
    if (rank <= 16) return f(std::integral_constant<int, 1>());
    if (rank <= 32) return f(std::integral_constant<int, 2>());
    if (rank <= 64) return f(std::integral_constant<int, 4>());
    return f(std::integral_constant<int, 8>());
}
// Parts of the output channels: until there are two workgroups a CU, `wide` channels (a block for each wave) at least.  More
// parts cost more first products than their balance gains: 16411 x 768 f32 channel-first 42 us, with up to 1200 workgroups 45.
int parts(int tiles, int cout, int wide) { return std::max(1, std::min((cout + wide - 1) / wide, 512 / std::max(1, tiles))); }

// 64 tokens a workgroup instead of 32, once that leaves two workgroups a CU: the factors are read half as often, which counts
// where there are more ranks than tokens of a tile.  65536 tokens 768 -> 768 bf16 rank 64 72 us (32 tokens: 87), rank 128 143
// (174), f32 rank 64 173 (194); with one rank tile 65536 tokens 768 -> 2048 243 (154), 16384 tokens rank 64 24 (20).
// The 32-bit offsets of such a tile reach its 64th row because at least 2^15 rows of that length lie in the card's memory:
// less than 2^24 bytes each.  (Of 32 rows they reach at the ld of 2^25 that the checks allow.)
template <class T, int RT> constexpr bool kLargeTiles = RT >= 4;
template <class T> hipError_t forward(const k82_lora& p, const std::vector<op::Seg>& segs, hipStream_t st, bool across = false) {
    return by_rank(p.rank, [&](auto rt) -> hipError_t {
        constexpr int RT = decltype(rt)::value, V = Vec<T>::N;
        const bool even = p.cin % V == 0 && p.cout % V == 0 && p.rank % V == 0;
        if constexpr (std::is_same<T, float>::value)
            if (p.layout == K82_COLS) {
                constexpr int NW = RT <= 2 ? 8 : 4;
                auto go = [&](auto tt) -> hipError_t {
                    constexpr int TT = decltype(tt)::value;
                    for (const SegTable& t : op::tables(segs, 16 * TT, true)) {
                        const int tiles = t.tile0[t.n];
                        OP_TRY(op::run(even ? lora_cols_kernel<NW, RT, TT, true> : lora_cols_kernel<NW, RT, TT, false>,
                                       dim3(tiles, parts(tiles, p.cout, 16 * NW)), dim3(64 * NW), 0, st, t, p));
                    }
                    return hipSuccess;
                };
                // pairs of tokens a lane (128 bytes of a channel a tile), where there is a pair
                return p.tokens >= 2 ? go(std::integral_constant<int, 2>()) : go(std::integral_constant<int, 1>());
            }
        auto go = [&](auto tt) -> hipError_t {
            constexpr int TT = decltype(tt)::value, NW = 4;
            for (const SegTable& t : op::tables(segs, 16 * TT)) {
                const int tiles = t.tile0[t.n];
                auto kernel = even ? lora_rows_kernel<T, NW, RT, TT, true> : lora_rows_kernel<T, NW, RT, TT, false>;
                if constexpr (RT == 1 && V == 4)
                    if (across) kernel = even ? lora_rows_kernel<T, NW, RT, TT, true, true> : lora_rows_kernel<T, NW, RT, TT, false, true>;
                OP_TRY(op::run(kernel, dim3(tiles, parts(tiles, p.cout, 8 * NW * V)), dim3(64 * NW), 0, st, t, p));
            }
            return hipSuccess;
        };
        if constexpr (kLargeTiles<T, RT>) {
            int64_t tokens = 0;
            for (const op::Seg& g : segs) tokens += g.len;
            if (!across && tokens >= 64 * 512) return go(std::integral_constant<int, 4>());
        }
        return go(std::integral_constant<int, 2>());
    });
}

// workgroups along the channels and rank shares of the weight's gradient (as lora_weight_kernel takes them apart)
int weight_groups(const k82_lora_grad& p) {
    const int shares = (p.rank + 31) / 32, pair = shares > 1 ? 2 : 1, per = kWaves / pair;
    return ((p.cin + 127) / 128 + (p.cout + 127) / 128 + per - 1) / per * ((shares + pair - 1) / pair);
}
// Tokens of a chunk of it: as many workgroups a CU as its registers let run at once, two (f32 of more than 16 ranks: three),
// once there are tokens for them; more would wait for them, and their partial sums are traffic.  The whole backward pass with 512
// workgroups and with 768: 65536 tokens 768 / 2048 bf16 rank 16 190 and 192 us, f32 rank 32 444 and 397; 32768 tokens 768 / 768
// bf16 rank 64 94 and 107; 8192 tokens bf16 rank 16 32 and 38.  (Against the rule: 65536 tokens f32 rank 16 394 and 366.)
int chunk_rows(const k82_lora_grad& p, int64_t tokens) {
    const int64_t chunks = std::max<int64_t>(1, (p.rank <= 16 || p.dtype == K82_BF16 ? 512 : 768) / weight_groups(p));
    return (int)std::max<int64_t>(32, ((tokens + chunks - 1) / chunks + 31) / 32 * 32);
}
// One rank tile in f32: the factors are read across instead of being transposed first, a launch less (211 tokens 768 -> 768 rank
// 7 23 us, transposed 28; 16384 tokens rank 16 66 and 67).  Not in bf16, eight loads for 16 bytes (16384 tokens 49 and 46), nor
// for more ranks (1024 tokens 768 -> 2048 f32 rank 64 107 and 82).
bool reads_across(const k82_lora_grad& p) { return p.dtype == K82_F32 && p.rank <= 16; }
struct Layout { int64_t g, at, bt, scale, part, end; };         // bytes
Layout layout(const k82_lora_grad& p, const k82_segments& s) {
    const int64_t size = p.dtype == K82_F32 ? 4 : 2, used = reads_across(p) ? 0 : std::min<int64_t>(s.n, p.adapters), all = (int64_t)p.cin + p.cout;
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
    std::vector<op::Seg> segs = op::merged(s);
    if (reads_across(p)) {
        const k82_lora f{p.dtype, K82_ROWS, K82_ACT_NONE, p.cout, p.cin, p.rank, p.adapters, p.tokens, p.dy, p.lddy,
                         p.dx_base, p.lddx_base, p.dx, p.lddx, p.b, p.a, p.scale, g};
        OP_TRY(forward<T>(f, segs, st, true));
    } else {
        // the adapters in use, numbered in the order of their index
        std::vector<int> used, number(p.adapters, -1);
        for (const RunTable& t : plan.tables)
            for (int i = 0; i < t.runs; ++i)
                if (number[t.index[i]] < 0) { number[t.index[i]] = (int)used.size(); used.push_back(t.index[i]); }
        const int64_t factor = (int64_t)p.rank;
        for (size_t i = 0; i < used.size(); i += op::kSegs) {
            Used u;
            u.n = (int)std::min<size_t>(op::kSegs, used.size() - i);
            std::copy_n(used.begin() + i, u.n, u.index);
            OP_TRY(op::run(lora_transpose_kernel<T>, dim3((p.cin + 31) / 32 + (p.cout + 31) / 32, (p.rank + 31) / 32, u.n), dim3(256), 0, st, u, p,
                           at + i * factor * p.cin, bt + i * factor * p.cout, scale + i));
        }
        for (op::Seg& v : segs)
            if (v.index >= 0) v.index = number[v.index];
        const k82_lora f{p.dtype, K82_ROWS, K82_ACT_NONE, p.cout, p.cin, p.rank, (int)used.size(), p.tokens, p.dy, p.lddy,
                         p.dx_base, p.lddx_base, p.dx, p.lddx, bt, at, scale, g};
        OP_TRY(forward<T>(f, segs, st));
    }
    const bool even = p.cin % Vec<T>::N == 0 && p.cout % Vec<T>::N == 0;
    for (const RunTable& t : plan.tables) {
        const auto kernel = p.rank <= 16 ? (even ? lora_weight_kernel<T, 1, true> : lora_weight_kernel<T, 1, false>)
                                         : (even ? lora_weight_kernel<T, 2, true> : lora_weight_kernel<T, 2, false>);
        OP_TRY(op::run(kernel, dim3(weight_groups(p), t.chunk0[t.runs] - t.chunk0[0]), dim3(64 * kWaves), 0, st, t, p, (const float*)g, part));
    }
    for (const ReduceTable& t : plan.reduce)
        OP_TRY(op::run(lora_reduce_kernel, dim3((p.cin + 63) / 64 + (p.cout + 63) / 64, (p.rank + 15) / 16, t.n), dim3(1024), 0, st, t, p.cin, p.cout, p.rank,
                       (const float*)part, p.da, p.db));
    return hipSuccess;
}
}  // namespace

namespace op {
int64_t workspace(const k82_lora_grad& p, const k82_segments& s) { return layout(p, s).end; }
hipError_t launch(const k82_lora& p, const k82_segments& s, hipStream_t st) {
    const std::vector<Seg> segs = merged(s);
    return p.dtype == K82_F32 ? forward<float>(p, segs, st) : forward<bf16_t>(p, segs, st);
}
hipError_t launch(const k82_lora_grad& p, const k82_segments& s, void* ws, hipStream_t st) {
    return p.dtype == K82_F32 ? backward<float>(p, s, ws, st) : backward<bf16_t>(p, s, ws, st);
}
}  // namespace op
