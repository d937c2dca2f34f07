// Argument checks and segment tables of the operators on caller-owned tensors (operators.h): host code, no GPU needed.
#include "operators.h"

#include <algorithm>

namespace op {
namespace {

// A tensor [outer][inner] with `ld` elements between rows of memory (K82_ROWS: outer = tokens, K82_COLS: channels)
struct Span {
    const char* p;
    int64_t row, outer, inner;                 // bytes, rows, bytes
    Span(const void* q, int64_t ld, int layout, int64_t tokens, int64_t c, int size)
        : p((const char*)q), row(ld * size), outer(layout == K82_COLS ? c : tokens),
          inner((layout == K82_COLS ? tokens : c) * size) {}
    int64_t bytes() const { return outer > 0 ? (outer - 1) * row + inner : 0; }
};
bool overlap(const Span& a, const Span& b) {
    if (!a.p || !b.p || a.bytes() == 0 || b.bytes() == 0) return false;
    if (a.p + a.bytes() <= b.p || b.p + b.bytes() <= a.p) return false;
    if (a.row == b.row && a.row > 0) {         // interleaved slices of one buffer
        const int64_t m = ((b.p - a.p) % a.row + a.row) % a.row;
        if (m >= a.inner && m + b.inner <= a.row) return false;
    }
    return true;
}
bool same(const Span& a, const Span& b) { return a.p == b.p && (a.row == b.row || a.outer <= 1); }

std::string check_segments(const k82_segments* s, int64_t tokens, int lo, int hi, const char* what) {
    if (!s) return "segments must not be NULL";
    if (s->n < 0) return "segments: n must not be negative";
    if (s->n == 0) return "";
    if (!s->off || !s->index) return "segments: off and index must not be NULL";
    if (s->off[0] < 0) return "segments: off[0] must not be negative";
    for (int32_t i = 0; i < s->n; ++i) {
        if (s->off[i + 1] < s->off[i]) return "segments: off must not decrease (at " + std::to_string(i) + ")";
        if ((s->index[i] < lo && s->index[i] != K82_SKIP) || s->index[i] >= hi)
            return std::string("segments: index ") + std::to_string(s->index[i]) + " of segment " + std::to_string(i) +
                   " is outside [" + std::to_string(lo) + ", " + what + " = " + std::to_string(hi) + ")";
    }
    if (s->off[s->n] > tokens)
        return "segments: off ends at " + std::to_string(s->off[s->n]) + ", the tensors hold " + std::to_string(tokens) + " tokens";
    return "";
}
std::string check_sizes(int dtype, int layout, int64_t tokens, std::initializer_list<int> channels) {
    if (dtype != K82_F32 && dtype != K82_BF16) return "dtype must be K82_F32 or K82_BF16";
    if (layout != K82_ROWS && layout != K82_COLS) return "layout must be K82_ROWS or K82_COLS";
    if (layout == K82_COLS && dtype != K82_F32) return "K82_COLS exists in K82_F32 only";
    // a launch may need 256 threads for a token and holds less than 2^32; every offset into a tensor is 64 bits wide
    if (tokens < 0 || tokens >= 1 << 24) return "tokens must be in [0, 2^24)";
    for (int c : channels)
        if (c < 1 || c > (1 << 20)) return "channel counts must be in [1, 2^20]";
    return "";
}
std::string check_tensor(const char* name, const void* p, int64_t ld, int layout, int64_t tokens, int64_t c, int size, bool optional) {
    if (!p) return optional || tokens == 0 ? "" : std::string(name) + " must not be NULL";
    if ((uintptr_t)p % size) return std::string(name) + " is not aligned to its element";
    if (ld < (layout == K82_COLS ? tokens : c)) return std::string("ld of ") + name + " is smaller than a row of it";
    if (ld > 1 << 25) return std::string("ld of ") + name + " is larger than 2^25";       // (offsets inside a tile of rows are 32 bits wide)
    return "";
}
std::string check_aligned(int size, std::initializer_list<const void*> p) {
    for (const void* v : p)
        if ((uintptr_t)v % size) return "a pointer is not aligned to its element";
    return "";
}
std::string check_lora_factors(int rank, int adapters, const void* a, const void* b, const float* scale) {
    if (rank < 1 || rank > K82_LORA_MAX_RANK) return "rank must be in [1, 128]";
    if (adapters < 0) return "adapters must not be negative";
    if (adapters > 0 && (!a || !b || !scale)) return "a, b and scale must not be NULL";
    return "";
}
#define OP_CHECK(e)                     \
    do {                                \
        const std::string m_ = (e);     \
        if (!m_.empty()) return m_;     \
    } while (0)

}  // namespace

std::string check(const k82_lora* p, const k82_segments* s) {
    if (!p) return "arguments must not be NULL";
    OP_CHECK(check_sizes(p->dtype, p->layout, p->tokens, {p->cin, p->cout}));
    OP_CHECK(check_lora_factors(p->rank, p->adapters, p->a, p->b, p->scale));
    if (p->act != K82_ACT_NONE && p->act != K82_ACT_GELU_NEW) return "act must be K82_ACT_NONE or K82_ACT_GELU_NEW";
    OP_CHECK(check_segments(s, p->tokens, -1, p->adapters, "adapters"));
    const int size = p->dtype == K82_F32 ? 4 : 2;
    OP_CHECK(check_tensor("x", p->x, p->ldx, p->layout, p->tokens, p->cin, size, false));
    OP_CHECK(check_tensor("base", p->base, p->ldbase, p->layout, p->tokens, p->cout, size, true));
    OP_CHECK(check_tensor("y", p->y, p->ldy, p->layout, p->tokens, p->cout, size, false));
    OP_CHECK(check_aligned(size, {p->a, p->b}));
    OP_CHECK(check_aligned(4, {p->scale, p->h}));
    const Span x(p->x, p->ldx, p->layout, p->tokens, p->cin, size), y(p->y, p->ldy, p->layout, p->tokens, p->cout, size),
        base(p->base, p->ldbase, p->layout, p->tokens, p->cout, size), h(p->h, p->rank, K82_ROWS, p->tokens, p->rank, 4);
    if (overlap(x, y)) return "x and y overlap";
    if (overlap(base, y) && !same(base, y)) return "base and y overlap without being one tensor";
    if (overlap(h, x) || overlap(h, y) || overlap(h, base)) return "h overlaps another tensor";
    return "";
}
std::string check(const k82_lora_grad* p, const k82_segments* s) {
    if (!p) return "arguments must not be NULL";
    OP_CHECK(check_sizes(p->dtype, K82_ROWS, p->tokens, {p->cin, p->cout}));
    OP_CHECK(check_lora_factors(p->rank, p->adapters, p->a, p->b, p->scale));
    if (p->adapters >= 1 << 24) return "adapters must be less than 2^24";       // (each has sums to be written, by numbers of 32 bits)
    if (p->adapters > 0 && (!p->da || !p->db)) return "da and db must not be NULL";
    OP_CHECK(check_segments(s, p->tokens, -1, p->adapters, "adapters"));
    const int size = p->dtype == K82_F32 ? 4 : 2;
    OP_CHECK(check_tensor("x", p->x, p->ldx, K82_ROWS, p->tokens, p->cin, size, false));
    OP_CHECK(check_tensor("dy", p->dy, p->lddy, K82_ROWS, p->tokens, p->cout, size, false));
    OP_CHECK(check_tensor("h", p->h, p->rank, K82_ROWS, p->tokens, p->rank, 4, false));
    OP_CHECK(check_tensor("dx_base", p->dx_base, p->lddx_base, K82_ROWS, p->tokens, p->cin, size, true));
    OP_CHECK(check_tensor("dx", p->dx, p->lddx, K82_ROWS, p->tokens, p->cin, size, false));
    OP_CHECK(check_aligned(size, {p->a, p->b}));
    OP_CHECK(check_aligned(4, {p->scale, p->h, p->da, p->db}));
    const Span x(p->x, p->ldx, K82_ROWS, p->tokens, p->cin, size), dx(p->dx, p->lddx, K82_ROWS, p->tokens, p->cin, size),
        dy(p->dy, p->lddy, K82_ROWS, p->tokens, p->cout, size), h(p->h, p->rank, K82_ROWS, p->tokens, p->rank, 4),
        base(p->dx_base, p->lddx_base, K82_ROWS, p->tokens, p->cin, size);
    if (overlap(dx, x) || overlap(dx, dy) || overlap(dx, h)) return "dx overlaps x, dy or h";
    if (overlap(base, dx) && !same(base, dx)) return "dx_base and dx overlap without being one tensor";
    return "";
}
std::string check(const k82_layernorm* p, const k82_segments* s) {
    if (!p) return "arguments must not be NULL";
    OP_CHECK(check_sizes(p->dtype, p->layout, p->tokens, {p->c}));
    if (p->gains < 1 || !p->gain || !p->offset) return "gain and offset must hold at least one row";
    if (!(p->eps >= 0.f)) return "eps must not be negative";
    if (!p->mean != !p->rstd) return "mean and rstd come together";
    OP_CHECK(check_segments(s, p->tokens, 0, p->gains, "gains"));
    const int size = p->dtype == K82_F32 ? 4 : 2;
    OP_CHECK(check_tensor("x", p->x, p->ldx, p->layout, p->tokens, p->c, size, false));
    OP_CHECK(check_tensor("res", p->res, p->ldres, p->layout, p->tokens, p->c, size, true));
    OP_CHECK(check_tensor("y", p->y, p->ldy, p->layout, p->tokens, p->c, size, false));
    OP_CHECK(check_aligned(size, {p->gain, p->offset}));
    OP_CHECK(check_aligned(4, {p->mean, p->rstd}));
    const Span x(p->x, p->ldx, p->layout, p->tokens, p->c, size), res(p->res, p->ldres, p->layout, p->tokens, p->c, size),
        y(p->y, p->ldy, p->layout, p->tokens, p->c, size), m(p->mean, 1, K82_ROWS, p->tokens, 1, 4), r(p->rstd, 1, K82_ROWS, p->tokens, 1, 4);
    if (overlap(x, y) && !same(x, y)) return "x and y overlap without being one tensor";
    if (overlap(res, y) && !same(res, y)) return "res and y overlap without being one tensor";
    if (overlap(m, r) || overlap(m, y) || overlap(r, y) || overlap(m, x) || overlap(r, x) || overlap(m, res) || overlap(r, res))
        return "mean or rstd overlaps another tensor";
    return "";
}
std::string check(const k82_layernorm_grad* p, const k82_segments* s) {
    if (!p) return "arguments must not be NULL";
    OP_CHECK(check_sizes(p->dtype, K82_ROWS, p->tokens, {p->c}));
    if (p->gains < 1 || !p->gain || !p->dgain || !p->doffset) return "gain, dgain and doffset must hold at least one row";
    if (p->gains >= 1 << 24) return "gains must be less than 2^24";
    if (p->tokens > 0 && (!p->mean || !p->rstd)) return "mean and rstd must not be NULL";
    OP_CHECK(check_segments(s, p->tokens, 0, p->gains, "gains"));
    const int size = p->dtype == K82_F32 ? 4 : 2;
    OP_CHECK(check_tensor("x", p->x, p->ldx, K82_ROWS, p->tokens, p->c, size, false));
    OP_CHECK(check_tensor("res", p->res, p->ldres, K82_ROWS, p->tokens, p->c, size, true));
    OP_CHECK(check_tensor("dy", p->dy, p->lddy, K82_ROWS, p->tokens, p->c, size, false));
    OP_CHECK(check_tensor("dx", p->dx, p->lddx, K82_ROWS, p->tokens, p->c, size, false));
    OP_CHECK(check_aligned(size, {p->gain}));
    OP_CHECK(check_aligned(4, {p->mean, p->rstd, p->dgain, p->doffset}));
    const Span dx(p->dx, p->lddx, K82_ROWS, p->tokens, p->c, size);
    const Span in[3] = {{p->x, p->ldx, K82_ROWS, p->tokens, p->c, size}, {p->res, p->ldres, K82_ROWS, p->tokens, p->c, size},
                        {p->dy, p->lddy, K82_ROWS, p->tokens, p->c, size}};
    for (const Span& v : in)
        if (overlap(v, dx) && !same(v, dx)) return "dx overlaps an input without being one tensor with it";
    const Span st[2] = {{p->mean, 1, K82_ROWS, p->tokens, 1, 4}, {p->rstd, 1, K82_ROWS, p->tokens, 1, 4}};
    for (const Span& v : st)
        if (overlap(v, dx)) return "dx overlaps mean or rstd";
    return "";
}

std::vector<Seg> merged(const k82_segments& s, bool walked) {
    std::vector<Seg> v;
    for (int32_t i = 0; i < s.n; ++i) {
        const int start = (int)s.off[i], len = (int)(s.off[i + 1] - s.off[i]);
        if (len == 0 || (s.index[i] == K82_SKIP && (!walked || v.empty()))) continue;
        if (!v.empty() && v.back().index == s.index[i] && v.back().start + v.back().len == start) v.back().len += len;
        else v.push_back({start, len, s.index[i]});
    }
    while (!v.empty() && v.back().index == K82_SKIP) v.pop_back();
    return v;
}
std::vector<SegTable> tables(const std::vector<Seg>& segs, int tile, bool grid) {
    std::vector<SegTable> out;
    for (size_t i0 = 0; i0 < segs.size(); i0 += kSegs) {
        out.emplace_back();
        SegTable& t = out.back();
        t.n = (int)std::min<size_t>(kSegs, segs.size() - i0);
        t.tile0[0] = 0;
        for (int i = 0; i < kSegs; ++i) {
            if (i < t.n) {
                const Seg& g = segs[i0 + i];
                t.start[i] = g.start; t.len[i] = g.len; t.index[i] = g.index;
                const int before = grid ? g.start % tile : 0;
                t.tile0[i + 1] = t.tile0[i] + (before + g.len - 1) / tile + 1;
            } else {
                t.start[i] = 0; t.len[i] = 0; t.index[i] = -1;
                t.tile0[i + 1] = t.tile0[t.n];
            }
        }
    }
    return out;
}

RunPlan runs(const k82_segments& s, int indices, int rows) {
    std::vector<Seg> v = merged(s);
    v.erase(std::remove_if(v.begin(), v.end(), [](const Seg& g) { return g.index < 0; }), v.end());
    std::stable_sort(v.begin(), v.end(), [](const Seg& a, const Seg& b) { return a.index < b.index; });
    RunPlan plan;
    std::vector<int> count(indices + 1, 0);    // chunks of each index
    for (size_t i0 = 0; i0 < v.size(); i0 += kSegs) {
        plan.tables.emplace_back();
        RunTable& t = plan.tables.back();
        t.pieces = (int)std::min<size_t>(kSegs, v.size() - i0);
        t.runs = 0; t.rows = rows;
        t.cum[0] = 0;
        for (int i = 0; i < t.pieces; ++i) {
            const Seg& g = v[i0 + i];
            if (i == 0 || g.index != t.index[t.runs - 1]) { t.index[t.runs] = g.index; t.run_cum[t.runs++] = t.cum[i]; }
            t.start[i] = g.start;
            t.cum[i + 1] = t.cum[i] + g.len;
        }
        t.run_cum[t.runs] = t.cum[t.pieces];
        t.chunk0[0] = plan.chunks;
        for (int r = 0; r < t.runs; ++r) {
            const int n = (t.run_cum[r + 1] - t.run_cum[r] - 1) / rows + 1;
            t.chunk0[r + 1] = t.chunk0[r] + n;
            count[t.index[r]] += n;
        }
        plan.chunks = t.chunk0[t.runs];
        for (int i = t.pieces; i < kSegs; ++i) { t.start[i] = 0; t.cum[i + 1] = t.cum[t.pieces]; }
        for (int i = t.runs; i < kSegs; ++i) { t.index[i] = 0; t.run_cum[i + 1] = t.run_cum[t.runs]; t.chunk0[i + 1] = t.chunk0[t.runs]; }
    }
    for (int b = 0, first = 0; b < indices; b += kSegs) {
        plan.reduce.emplace_back();
        ReduceTable& t = plan.reduce.back();
        t.base = b;
        t.n = std::min(kSegs, indices - b);
        t.first[0] = first;
        for (int i = 0; i < kSegs; ++i) t.first[i + 1] = t.first[i] + (i < t.n ? count[b + i] : 0);
        first = t.first[t.n];
    }
    return plan;
}

}  // namespace op
