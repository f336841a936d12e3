// Host: do an operator's outputs share memory with its inputs or with each other? Tensors are rows of contiguous bytes under up
// to two strides; halves of one buffer interleave without sharing anything, so spans alone do not tell.
#pragma once
#include <algorithm>
#include <initializer_list>

// rows of `row` bytes at `at` + i s[0] + j s[1], i < n[0], j < n[1]; row = 0: no tensor
struct View {
    long long at, row, n[2], s[2];
    View() : at(0), row(0), n{1, 1}, s{0, 0} {}
    View(const void* q, long long bytes) : View(q, bytes, 1, 0, 1, 0) {}
    View(const void* q, long long row, long long n0, long long s0, long long n1 = 1, long long s1 = 0)
        : at((long long)q), row(q ? row : 0), n{n0, n1}, s{s0, s1} {}
    long long end() const { return at + row + (n[0] - 1) * s[0] + (n[1] - 1) * s[1]; }
};

// One stride of the difference between two addresses: x s, lo <= x <= hi
struct Term { long long s, lo, hi; };

inline long long floor_div(long long a, long long b) { return a / b - (a % b != 0 && a < 0); }        // b > 0

// is there a sum base + x_0 s_0 + ... strictly between lo and hi? Larger strides first: in nested layouts one or two x a level
// remain. Where the search takes long (four strides that nest in no order) the answer is yes.
inline bool reaches(const Term* t, int n, long long base, long long lo, long long hi, int& left) {
    if (n == 0) return lo < base && base < hi;
    long long rest_lo = 0, rest_hi = 0;
    for (int k = 1; k < n; ++k) { rest_lo += t[k].lo * t[k].s; rest_hi += t[k].hi * t[k].s; }
    const long long x0 = std::max(t->lo, floor_div(lo - base - rest_hi, t->s) + 1), x1 = std::min(t->hi, floor_div(hi - base - rest_lo - 1, t->s));
    if (n == 1) return x0 <= x1;
    for (long long x = x0; x <= x1; ++x) {
        if (--left < 0) return true;
        if (reaches(t + 1, n - 1, base + x * t->s, lo, hi, left)) return true;
    }
    return false;
}

inline bool share(const View& a, const View& b) {
    if (!a.row || !b.row || a.end() <= b.at || b.end() <= a.at) return false;
    Term t[4];
    int n = 0;
    const auto add = [&](long long s, long long lo, long long hi) {
        if (s == 0 || lo == hi) return;
        for (int k = 0; k < n; ++k) if (t[k].s == s) { t[k].lo += lo; t[k].hi += hi; return; }
        t[n++] = {s, lo, hi};
    };
    for (int k = 0; k < 2; ++k) { add(a.s[k], 0, a.n[k] - 1); add(b.s[k], 1 - b.n[k], 0); }
    std::sort(t, t + n, [](const Term& x, const Term& y) { return x.s > y.s; });
    int left = 1 << 16;
    return reaches(t, n, a.at - b.at, -a.row, b.row, left);
}

inline bool apart(const View* out, int n_out, const View* in, int n_in) {
    for (int i = 0; i < n_out; ++i) {
        for (int k = i + 1; k < n_out; ++k) if (share(out[i], out[k])) return false;
        for (int k = 0; k < n_in; ++k) if (share(out[i], in[k])) return false;
    }
    return true;
}
inline bool apart(std::initializer_list<View> out, std::initializer_list<View> in) {
    return apart(out.begin(), (int)out.size(), in.begin(), (int)in.size());
}
