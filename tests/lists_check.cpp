// Host side of the operators over lists of tensors (csrc/grads_lists.h) against brute force: overlaps of written memory, and the tables of the
// launches -- every double of every tensor in exactly one chunk, every address as given, wherever the tensors lie.
#include "grads_lists.h"
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>

#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); exit(1); } } while (0)
std::mt19937_64 rng(1);

void overlaps() {
    for (int it = 0; it < 20000; ++it) {
        const int nt = 1 + rng() % 4, unit = 1 + rng() % 2, mode = rng() % 3, NP = mode == 1 ? 3 : 2;      // mode: clip, momentum step, step
        const double* p[3][4];
        long long n[4];
        for (int i = 0; i < nt; ++i) {
            n[i] = rng() % 6;
            for (int j = 0; j < 3; ++j) p[j][i] = (const double*)(uintptr_t)(8 * (100 + rng() % 150));
            if (mode == 0 && rng() % 2) p[1][i] = p[0][i];
        }
        const bool w[3] = {mode != 0, mode == 0, mode == 1};
        bool bad = false;
        for (int a = 0; a < NP; ++a)
            for (int i = 0; i < nt; ++i)
                for (int b = 0; b < NP && w[a]; ++b)
                    for (int j = 0; j < nt; ++j) {
                        if ((a == b && i == j) || (mode == 0 && i == j && p[a][i] == p[b][j]) || !n[i] || !n[j]) continue;
                        bad |= p[a][i] < p[b][j] + unit * n[j] && p[b][j] < p[a][i] + unit * n[i];
                    }
        const bool clip[2] = {false, true}, step3[3] = {true, false, true}, step2[2] = {true, false};
        const std::string e = mode == 0 ? check_lists(Lists<2>{nt, {p[0], p[1]}, n, unit}, clip, 1)
                            : mode == 1 ? check_lists(Lists<3>{nt, {p[0], p[1], p[2]}, n, unit}, step3, 0)
                                        : check_lists(Lists<2>{nt, {p[0], p[1]}, n, unit}, step2, 0);
        CHECK(e.empty() != bad);
    }
}

template <int NP> void tables() {
    for (int it = 0; it < 240; ++it) {
        const int nt = 1 + rng() % (it % 8 ? 60 : 900), chunk = it & 1 ? PIECE : CHUNK, unit = 1 + (it >> 1) % 2, spread = it % 5;
        std::vector<long long> n(nt);
        std::vector<const double*> x[NP];
        for (auto& v : n) {
            const int k = rng() % 6;
            v = k == 0 ? 0 : k == 1 ? rng() % 10 : k == 2 ? chunk - 2 + rng() % 5 : k == 3 ? 2 * chunk - 2 + rng() % 5 : rng() % 50000;
        }
        for (int j = 0; j < NP; ++j)
            for (int i = 0; i < nt; ++i) {
                // all near each other; in few windows of 32 GB; in many; anywhere; near the lowest addresses
                const uintptr_t far = spread == 1 ? (uintptr_t)(i % 3) << 35 : spread == 2 ? (uintptr_t)(rng() % 40) << 36 : spread == 3 ? (rng() >> 17) & ~(uintptr_t)7 : 0;
                x[j].push_back((const double*)(far + ((uintptr_t)(spread == 4 ? 1 : 0x7f) << (spread == 4 ? 3 : 40)) + ((uintptr_t)(i * NP + j) << 20)));
            }
        Lists<NP> L{nt, {}, n.data(), unit};
        for (int j = 0; j < NP; ++j) L.p[j] = x[j].data();
        int launches = 0, full = 0;
        for (int i = 0; i < nt; ++launches) {
            Table<NP> t;
            memset((void*)&t, 0x5a, sizeof t);           // (what a stack holds)
            const int from = i;
            i = fill(L, i, t, chunk);
            CHECK(i > from && i <= nt);
            const unsigned G = t.first[t.N];
            unsigned q = 0;
            int k = 0;
            for (int e = from; e < i; ++e) {             // the tensors of the launch in their order
                if (!n[e]) continue;
                CHECK(k < t.N && t.first[k] == q && t.first[k + 1] > q);
                const long long len = (long long)(t.first[k + 1] - t.first[k] - 1) * chunk + t.tail[k] + 1;
                CHECK(len == n[e] * unit);
                for (int j = 0; j < NP; ++j) {
                    const double* a = (const double*)((uintptr_t)t.base[j][(t.which[k] >> (2 * j)) & 3] + 8 * (uintptr_t)t.offset[j][k]);
                    CHECK(a == x[j][e]);
                }
                q = t.first[++k];
            }
            CHECK(q == G);
            for (int e = k; e <= t.N; ++e) CHECK(t.first[e] == G);
            full += k == t.N;
        }
        CHECK(launches <= nt / 4 + 1);
        if (spread == 0 || spread == 1 || spread == 4) CHECK(launches <= full + 1);
    }
}

int main() {
    overlaps();
    tables<1>();
    tables<2>();
    tables<3>();
    // what is refused
    const bool w[1] = {false};
    const double* p[2] = {(const double*)64, (const double*)128};
    long long n[2] = {4, 4};
    CHECK(check_lists(Lists<1>{2, {p}, n, 1}, w, 0).empty() && check_lists(Lists<1>{0, {nullptr}, nullptr, 1}, w, 0).empty());
    CHECK(!check_lists(Lists<1>{-1, {p}, n, 1}, w, 0).empty() && !check_lists(Lists<1>{2, {nullptr}, n, 1}, w, 0).empty());
    CHECK(!check_lists(Lists<1>{2, {p}, nullptr, 1}, w, 0).empty());
    n[1] = -1;
    CHECK(!check_lists(Lists<1>{2, {p}, n, 1}, w, 0).empty());
    n[1] = (1LL << 40) + 1;
    CHECK(!check_lists(Lists<1>{2, {p}, n, 1}, w, 0).empty());
    n[0] = n[1] = 1LL << 40;
    CHECK(!check_lists(Lists<1>{2, {p}, n, 1}, w, 0).empty());
    n[0] = n[1] = 4;
    p[1] = nullptr;
    CHECK(!check_lists(Lists<1>{2, {p}, n, 1}, w, 0).empty());
    n[1] = 0;
    CHECK(check_lists(Lists<1>{2, {p}, n, 1}, w, 0).empty());
    p[1] = (const double*)132;
    n[1] = 4;
    CHECK(!check_lists(Lists<1>{2, {p}, n, 1}, w, 0).empty());
    printf("ok\n");
}
