// Host side of the operators over lists of tensors (grads.hip): the checks of a call's lists and the tables that its launches carry.  Plain C++.
#pragma once
#include <algorithm>
#include <cstdint>
#include <string>
#include <vector>

namespace {

constexpr int THREADS = 256;
constexpr int UNROLL = 4;              // 16-byte loads in flight per thread (545 MB: norms 87 us; 2: 97, 8: 91; 1.1 GB clipped 533; 2: 605, 8: 574)
constexpr int CHUNK = 2 * THREADS * UNROLL;      // doubles: what a workgroup takes at a time; a chunk lies in one tensor
constexpr int PIECE = 128;             // doubles: what a wave takes at a time in the one-workgroup kernels
constexpr int WS_HEAD = 4;             // ws: N2, Ninf, c, what the kernels multiply by, then the partial results (4 doubles each)
constexpr int PARTIALS = 1024, PARTIALS_LEAST = 64;      // workgroups of the norm pass: over all launches, and of each launch besides (512: 94 us)

// The tensors of one launch.  Their table travels by value in the kernel arguments (no host-to-device copy, so a call may be captured), which hold
// 4 kB: addresses are 32-bit counts of doubles above one of four bases (windows of 32 GB; an allocator's segments lie far apart), lengths what the
// last chunk holds.  More tensors per launch, fewer launches: each costs >= 4 us, more than the work on a hundred short tensors.
constexpr int BASES = 4;
template <int NP> struct Table {
    static constexpr int N = NP == 1 ? 320 : NP == 2 ? 256 : 192;
    double* base[NP][BASES];
    unsigned offset[NP][N];
    unsigned first[N + 1];             // chunks before tensor t; entries behind the last tensor hold the total
    unsigned short tail[N];            // doubles of the last chunk, less one (a complex element counts two)
    unsigned char which[N];            // bits 2 j, 2 j + 1: the base of list j
};
static_assert(sizeof(Table<1>) <= 3968 && sizeof(Table<2>) <= 3968 && sizeof(Table<3>) <= 3968, "the kernel arguments hold 4 kB");

// A list of nt tensors with NP pointers each
template <int NP> struct Lists {
    int nt; const double* const* p[NP]; const long long* n; long long unit;      // unit: doubles per element
};

// What is wrong with the lists of a call (empty: nothing): lengths, pointers and the memory that is written -- no written range may overlap any other
// range of the call (in a clip the range that is read and written under the same index may be one and the same).
template <int NP> std::string check_lists(const Lists<NP>& L, const bool (&written)[NP], int same_as_first) {
    if (L.nt < 0) return "negative number of tensors";
    if (L.nt && !L.n) return "lengths missing";
    for (int j = 0; j < NP; ++j) if (L.nt && !L.p[j]) return "pointers missing";
    long long total = 0;
    bool any_written = false;
    for (int i = 0; i < L.nt; ++i) {
        if (L.n[i] < 0 || L.n[i] > (1LL << 40)) return "length of tensor " + std::to_string(i) + " out of range";
        total += L.n[i];
        if (total > (1LL << 40)) return "list too long";
        if (!L.n[i]) continue;
        for (int j = 0; j < NP; ++j) {
            if (!L.p[j][i]) return "null pointer for tensor " + std::to_string(i);
            if ((uintptr_t)L.p[j][i] % 8) return "tensor " + std::to_string(i) + " is not aligned to 8 bytes";
        }
    }
    for (int j = 0; j < NP; ++j) any_written |= written[j];
    if (!any_written) return {};
    struct Range { uintptr_t a, b; bool w; };
    std::vector<Range> r;
    r.reserve((size_t)NP * L.nt);
    for (int i = 0; i < L.nt; ++i)
        for (int j = 0; j < NP; ++j) {
            if (!L.n[i] || (j > 0 && j == same_as_first && L.p[j][i] == L.p[0][i])) continue;
            const uintptr_t a = (uintptr_t)L.p[j][i];
            const bool w = written[j] || (j == 0 && same_as_first > 0 && L.p[same_as_first][i] == L.p[0][i]);
            r.push_back({a, a + (uintptr_t)(8 * L.unit * L.n[i]), w});
        }
    std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.a < y.a; });
    uintptr_t end_any = 0, end_written = 0;
    for (const Range& x : r) {
        if (x.a < end_written || (x.w && x.a < end_any)) return "a tensor that is written overlaps another tensor of the call";
        if (x.b > end_any) end_any = x.b;
        if (x.w && x.b > end_written) end_written = x.b;
    }
    return {};
}

// The next launch's table from tensor `i` on; returns the index behind its last tensor.
template <int NP> int fill(const Lists<NP>& L, int i, Table<NP>& t, int chunk = CHUNK) {
    constexpr uintptr_t SPAN = (uintptr_t)8 << 32;       // what 32-bit counts of doubles reach
    int k = 0, bases[NP] = {};
    unsigned q = 0;
    for (; i < L.nt && k < t.N; ++i) {
        if (!L.n[i]) continue;
        int which[NP];
        bool fits = true;
        for (int j = 0; j < NP; ++j) {
            const uintptr_t x = (uintptr_t)L.p[j][i];
            int w = 0;
            while (w < bases[j] && x - (uintptr_t)t.base[j][w] >= SPAN) ++w;          // (an address below the base wraps round)
            which[j] = w;
            fits &= w < BASES;
        }
        if (!fits) break;                                // (never among the first four tensors)
        for (int j = 0; j < NP; ++j)
            if (which[j] == bases[j]) {
                const uintptr_t x = (uintptr_t)L.p[j][i];
                t.base[j][bases[j]++] = (double*)(x > SPAN / 2 ? x - SPAN / 2 : x % 8);
            }
        const long long n = L.n[i] * L.unit, c = (n + chunk - 1) / chunk;
        t.which[k] = 0;
        for (int j = 0; j < NP; ++j) {
            t.which[k] |= (unsigned char)(which[j] << (2 * j));
            t.offset[j][k] = (unsigned)(((uintptr_t)L.p[j][i] - (uintptr_t)t.base[j][which[j]]) / 8);
        }
        t.first[k] = q;
        t.tail[k++] = (unsigned short)(n - (c - 1) * chunk - 1);
        q += (unsigned)c;
    }
    for (int e = k; e <= t.N; ++e) t.first[e] = q;
    return i;
}

// What the choice of a kernel goes by: chunks and bytes of the list, whether one workgroup takes all of it
struct Size { unsigned chunks; int tensors; long long pieces, bytes; };
Size size_of(const long long* n, int nt, long long unit) {
    Size s{0, 0, 0, 0};
    for (int i = 0; i < nt; ++i) {
        const long long d = n[i] * unit;
        s.chunks += (unsigned)((d + CHUNK - 1) / CHUNK);
        s.pieces += (d + PIECE - 1) / PIECE;
        s.tensors += d > 0;
        s.bytes += 8 * d;
    }
    return s;
}
}  // namespace
