// overlap.h - do two strided pieces of memory share bytes?  Host code: the entry points of decay_attn.hip and layer_norm.hip
// refuse outputs that overlap each other or what is still read, also where rows are slices of one packed buffer and lie
// between each other's.
//
// Index vectors i of a and j of b meet where  -width_b < (b - a) + sum_d j_d s_d - i_d s_d < width_a.  Every index difference
// is bounded, so with the strides in falling order each term leaves few values by which the terms below it can still reach
// that window: one or two for nested layouts (a row inside a step inside a lane).  Layouts that would take more than TRIES
// values in all are counted as overlapping.
#pragma once
#include <cstdint>

namespace overlap {

struct Bytes {   // [at + sum_d i_d stride_d, + width), 0 <= i_d < count_d
    const void* at = nullptr;
    int64_t width = 0;
    int n = 0;
    struct { int64_t count, stride; } dim[3] = {};
    Bytes() {}
    Bytes(const void* p, int64_t bytes) : at(p), width(bytes) {}
    Bytes& by(int64_t count, int64_t stride) {
        dim[n].count = count;
        dim[n++].stride = stride;
        return *this;
    }
    bool empty() const {
        bool none = !at || width <= 0;
        for (int d = 0; d < n; d++) none = none || dim[d].count <= 0;
        return none;
    }
};

typedef __int128 Wide;   // (strides times counts pass 64 bits)
constexpr int TRIES = 1 << 16;

struct Terms {
    struct Term { Wide s; Wide lo, hi; } t[6];   // x s, lo <= x <= hi, s > 0, falling
    int n = 0;
    void add(Wide s, Wide lo, Wide hi, bool join) {
        if (s < 0) {
            const Wide l = lo;
            s = -s;
            lo = -hi;
            hi = -l;
        }
        int at = 0;
        while (at < n && t[at].s > s) at++;
        if (join && at < n && t[at].s == s) {
            t[at].lo += lo;
            t[at].hi += hi;
            return;
        }
        for (int i = n++; i > at; i--) t[i] = t[i - 1];
        t[at] = {s, lo, hi};
    }
};
inline Wide floor_div(Wide a, Wide b) { return a / b - (a % b < 0); }

// can the terms from k on add up to lo .. hi?  nonzero: not with every x zero
inline bool reaches(const Terms& m, int k, Wide lo, Wide hi, bool nonzero, int& tries) {
    if (k == m.n) return !nonzero && lo <= 0 && 0 <= hi;
    Wide below = 0, above = 0;
    for (int i = k + 1; i < m.n; i++) {
        below += m.t[i].s * m.t[i].lo;
        above += m.t[i].s * m.t[i].hi;
    }
    const auto& t = m.t[k];
    Wide x = -floor_div(above - lo, t.s), last = floor_div(hi - below, t.s);
    if (x < t.lo) x = t.lo;
    if (last > t.hi) last = t.hi;
    for (; x <= last; x++)
        if (--tries < 0 || reaches(m, k + 1, lo - x * t.s, hi - x * t.s, nonzero && x == 0, tries)) return true;
    return false;
}

inline bool meet(const Bytes& a, const Bytes& b) {
    if (a.empty() || b.empty()) return false;
    Terms m;
    for (int d = 0; d < a.n; d++)
        if (a.dim[d].count > 1 && a.dim[d].stride) m.add(a.dim[d].stride, 1 - a.dim[d].count, 0, true);
    for (int d = 0; d < b.n; d++)
        if (b.dim[d].count > 1 && b.dim[d].stride) m.add(b.dim[d].stride, 0, b.dim[d].count - 1, true);
    const Wide apart = (Wide)(uintptr_t)b.at - (Wide)(uintptr_t)a.at;
    int tries = TRIES;
    return reaches(m, 0, 1 - b.width - apart, a.width - 1 - apart, false, tries);
}

// two of its indexes share bytes
inline bool meets_itself(const Bytes& a) {
    if (a.empty()) return false;
    Terms m;
    for (int d = 0; d < a.n; d++)
        if (a.dim[d].count > 1) {
            if (!a.dim[d].stride) return true;
            m.add(a.dim[d].stride, 1 - a.dim[d].count, a.dim[d].count - 1, false);
        }
    int tries = TRIES;
    return reaches(m, 0, 1 - a.width, a.width - 1, true, tries);
}

// outputs that overlap themselves, each other or an input
template <int NO, int NI>
bool clash(const Bytes (&out)[NO], const Bytes (&in)[NI]) {
    for (int i = 0; i < NO; i++) {
        if (meets_itself(out[i])) return true;
        for (int j = i + 1; j < NO; j++)
            if (meet(out[i], out[j])) return true;
        for (int j = 0; j < NI; j++)
            if (meet(out[i], in[j])) return true;
    }
    return false;
}

}  // namespace overlap
