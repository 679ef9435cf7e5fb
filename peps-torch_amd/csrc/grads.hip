// The optimiser's operators over a LIST of tensors: 2-norm and largest modulus of the whole list, scaling to a bound of one of them, momentum
// step with that scaling in its registers (include/ctm_hip.h: ctm_grad_norms, ctm_grad_clip, ctm_sgd_step).
//
//   N2 = (sum_t sum_i |x_ti|^2)^1/2,  Ninf = max |x_ti|,  c = 1 if N <= max_norm else max_norm / N,
//   clip  y = c x          step  g' = c g,  m <- mu m + (1 - tau) g'  (first step: m <- g'),  p <- p - lr m
//
// All of it is bound by memory traffic on long lists (3 ... 9 flop per 8 ... 40 bytes) and by launches on short ones.  Nothing is kept between
// calls, nothing is read back by the host, no atomics and no memset: every sum has a fixed order, and a captured call replays as it ran.
#include "ctm_common.h"
#include <algorithm>

namespace {

constexpr int THREADS = 256;
constexpr int UNROLL = 4;              // 16-byte loads in flight per thread
constexpr int CHUNK = 2 * THREADS * UNROLL;      // doubles: what a workgroup takes at a time; a chunk lies in one tensor
constexpr int WS_HEAD = 4;             // ws: N2, Ninf, c, unused, then the partial results (4 doubles each)
constexpr int PARTIALS = 1024;         // workgroups of the norm pass over all launches, up to one more per launch

// The tensors of one launch.  Their table travels by value in the kernel arguments (no host-to-device copy, so a call may be captured), which hold
// 4 kB: addresses are 32-bit counts of doubles above the lowest one (tensors of a launch lie within 32 GB), lengths what the last chunk holds.
// More tensors per launch, fewer launches -- each costs >= 4 us, more than the work on a hundred short tensors.
template <int NP> struct Table {
    static constexpr int N = NP == 1 ? 384 : NP == 2 ? 256 : 192;
    double* base[NP];
    unsigned offset[NP][N];
    unsigned first[N + 1];             // chunks before tensor t; entries behind the last tensor hold the total
    unsigned short tail[N];            // doubles of the last chunk, less one (a complex element counts two)
};
static_assert(sizeof(Table<1>) <= 3968 && sizeof(Table<2>) <= 3968 && sizeof(Table<3>) <= 3968, "the kernel arguments hold 4 kB");

typedef double d2 __attribute__((ext_vector_type(2)));
typedef d2 d2u __attribute__((aligned(8)));          // 16-byte access at 8-byte alignment: views into a flat buffer start anywhere

template <bool NT> __device__ __forceinline__ d2 load2(const double* x) {
    if (NT) return __builtin_nontemporal_load((const d2u*)x);
    return *(const d2u*)x;
}
template <bool NT> __device__ __forceinline__ void store2(double* x, d2 v) {
    if (NT) __builtin_nontemporal_store((d2u)v, (d2u*)x);
    else *(d2u*)x = v;
}

// The tensor that holds chunk q: each lane of a wave compares N / 64 table entries, the count of those at or below q is its number.  The tensor
// found last is tried first: chunks of long tensors need no lookup.
template <int NP> struct Finder {
    static constexpr int R = Table<NP>::N / 64;
    const Table<NP>& t;
    unsigned mine[R];
    unsigned f = 0, l = 0;             // chunks of the tensor: f ... l - 1
    long long n = 0;                   // its doubles
    double* p[NP] = {};
    __device__ __forceinline__ explicit Finder(const Table<NP>& table) : t(table) {
#pragma unroll
        for (int j = 0; j < R; ++j) mine[j] = t.first[64 * j + (threadIdx.x & 63) + 1];
    }
    __device__ __forceinline__ void find(unsigned q, int chunk) {
        if (q >= f && q < l) return;
        int k = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) k += __popcll(__ballot(mine[j] <= q));
        k = __builtin_amdgcn_readfirstlane(k);
        f = t.first[k];
        l = t.first[k + 1];
        n = (long long)(l - f - 1) * chunk + t.tail[k] + 1;
#pragma unroll
        for (int j = 0; j < NP; ++j) p[j] = t.base[j] + t.offset[j][k];
    }
};

// Runs body(pointers, first double, length of the tensor) over this workgroup's chunks: every gridDim.x-th one, so that all workgroups sweep the
// list together (measured on 545 MB: 87 us for the norm pass against 95 with one contiguous share per workgroup, 185 against 223 for the
// scaling).  REVERSE: from the list's end to its beginning -- a second pass meets first what the pass before it left in the 256 MB last-level cache.
template <int NP, bool REVERSE, class F> __device__ __forceinline__ void chunks(const Table<NP>& t, F&& body) {
    Finder<NP> at(t);
    const unsigned G = t.first[Table<NP>::N];
    for (unsigned c = blockIdx.x; c < G; c += gridDim.x) {
        const unsigned q = REVERSE ? G - 1 - c : c;
        at.find(q, CHUNK);
        body(at.p, (long long)(q - at.f) * CHUNK, at.n);
    }
}

// Elements a + 2 u THREADS (+ 1) of this thread, zero behind the end of the tensor
template <bool NT> __device__ __forceinline__ void load_chunk(d2 (&v)[UNROLL], const double* x, long long a, long long n) {
    const long long i = a + 2 * threadIdx.x;
    if (a + CHUNK <= n) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) v[u] = load2<NT>(x + i + u * 2 * THREADS);
    } else {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const long long j = i + u * 2 * THREADS;
            v[u] = d2{0.0, 0.0};
            if (j + 1 < n) v[u] = load2<NT>(x + j);
            else if (j < n) v[u].x = x[j];               // (real tensors of odd length)
        }
    }
}
template <bool NT> __device__ __forceinline__ void store_chunk(const d2 (&v)[UNROLL], double* x, long long a, long long n) {
    const long long i = a + 2 * threadIdx.x;
    if (a + CHUNK <= n) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) store2<NT>(x + i + u * 2 * THREADS, v[u]);
    } else {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const long long j = i + u * 2 * THREADS;
            if (j + 1 < n) store2<NT>(x + j, v[u]);
            else if (j < n) x[j] = v[u].x;
        }
    }
}

// Sum of squares in three ranges (J. L. Blue, ACM TOMS 4 (1978) 15): elements between 2^-480 and 2^480 are squared as they are, the others scaled
// by 2^600 or 2^-600 first, so that neither overflow nor underflow of a square changes the norm.  The largest modulus is kept as the bit pattern
// of a non-negative double: the order of the patterns is that of the numbers, with NaN behind infinity, so a NaN survives the maximum.
struct Acc {
    double big = 0.0, med = 0.0, small = 0.0;
    unsigned long long top = 0;        // real: max |x|;  complex: max |z|^2 of the middle range
    unsigned long long top_far = 0;    // complex: max |z| of the others
};

__device__ __forceinline__ unsigned long long bits(double x) { return (unsigned long long)__double_as_longlong(x); }
__device__ __forceinline__ unsigned long long umax(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
constexpr unsigned EXP_LO = 1023 - 480, EXP_SPAN = 960;
__device__ __forceinline__ bool middle(double x) { return (((unsigned)__double2hiint(x) >> 20) & 0x7ffu) - EXP_LO < EXP_SPAN; }

__device__ __forceinline__ void add_far(Acc& a, double x) {
    const unsigned e = ((unsigned)__double2hiint(x) >> 20) & 0x7ffu;
    if (e >= EXP_LO + EXP_SPAN) { const double s = x * 0x1p-600; a.big = fma(s, s, a.big); }
    else if (e >= EXP_LO) a.med = fma(x, x, a.med);
    else { const double s = x * 0x1p600; a.small = fma(s, s, a.small); }
}

template <bool CPLX> __device__ __forceinline__ void add(Acc& a, d2 v) {
    // (zeros take the short way too: the imaginary parts of real data, masked entries)
    if ((middle(v.x) || v.x == 0.0) && (middle(v.y) || v.y == 0.0)) {
        const double s = fma(v.x, v.x, v.y * v.y);
        a.med += s;
        if (CPLX) a.top = umax(a.top, bits(s));
    } else {
        add_far(a, v.x);
        add_far(a, v.y);
        if (CPLX) a.top_far = umax(a.top_far, bits(hypot(v.x, v.y)));
    }
    if (!CPLX) { a.top = umax(a.top, bits(fabs(v.x))); a.top = umax(a.top, bits(fabs(v.y))); }
}

struct Part { double big, med, small; unsigned long long top; };

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

__device__ __forceinline__ void join(Part& p, const Part& q) {
    p.big += q.big; p.med += q.med; p.small += q.small; p.top = umax(p.top, q.top);
}

// Result of a workgroup of `WAVES` waves, the same bits on all its threads.
template <int WAVES> __device__ __forceinline__ Part reduce_block(Part p) {
    __shared__ Part sh[WAVES];
    p.med = wave_sum(p.med);
    if (__any(p.big != 0.0)) p.big = wave_sum(p.big);          // (true for NaN)
    if (__any(p.small != 0.0)) p.small = wave_sum(p.small);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) p.top = umax(p.top, __shfl_xor(p.top, o));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = p;
    __syncthreads();
    Part r = sh[0];
#pragma unroll 3                   // (not all 16 parts in registers at once, next to the list that small_kernel keeps there)
    for (int w = 1; w < WAVES; ++w) join(r, sh[w]);
    return r;
}

template <bool CPLX> __device__ __forceinline__ Part part_of(const Acc& a) {
    Part p{a.big, a.med, a.small, a.top};
    if (CPLX) p.top = umax(bits(sqrt(__longlong_as_double((long long)a.top))), a.top_far);
    return p;
}

struct Bound { double max_norm; int inf_norm; };      // max_norm < 0: no bound

// N2, Ninf and the factor c from the three range sums
struct Norms { double n2, ninf, c; };
__device__ __forceinline__ Norms finish(const Part& p, Bound bd) {
    Norms r;
    if (p.big != 0.0) r.n2 = sqrt(fma(p.med * 0x1p-600, 0x1p-600, p.big)) * 0x1p600;
    else if (p.med != 0.0) r.n2 = sqrt(fma(p.small * 0x1p-600, 0x1p-600, p.med));
    else r.n2 = sqrt(p.small) * 0x1p-600;
    r.ninf = __longlong_as_double((long long)p.top);
    const double n = bd.inf_norm ? r.ninf : r.n2;
    r.c = (bd.max_norm < 0.0 || n <= bd.max_norm) ? 1.0 : bd.max_norm / n;      // NaN norm: NaN
    return r;
}
__device__ __forceinline__ void put_norms(const Norms& r, double* ws) { ws[0] = r.n2; ws[1] = r.ninf; ws[2] = r.c; }

// First pass: partial results of the workgroups.
template <bool CPLX, bool NT>
__global__ __launch_bounds__(THREADS) void norm_partials_kernel(const Table<1> t, Part* out) {
    Acc acc;
    chunks<1, false>(t, [&](double* const* p, long long a, long long n) {
        d2 v[UNROLL];
        load_chunk<NT>(v, p[0], a, n);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) add<CPLX>(acc, v[u]);
    });
    const Part p = reduce_block<THREADS / 64>(part_of<CPLX>(acc));
    if (threadIdx.x == 0) out[blockIdx.x] = p;
}

// Norms from the partial results, by a workgroup of T threads, in an order that depends on T and np alone
template <int T> __device__ __forceinline__ Norms join_partials(const Part* part, int np, Bound bd) {
    Part p{0.0, 0.0, 0.0, 0};
    for (int i = threadIdx.x; i < np; i += T) join(p, part[i]);
    return finish(reduce_block<T / 64>(p), bd);
}

__global__ __launch_bounds__(1024) void norm_finish_kernel(const Part* part, int np, Bound bd, double* ws) {
    const Norms r = join_partials<1024>(part, np, bd);
    if (threadIdx.x == 0) put_norms(r, ws);
}

// Where the second pass gets its factor from: every workgroup joins the partial results by itself (32 kB at most, from the L2 cache; all get the
// same bits), which is cheaper than a kernel in between.
struct Source { const Part* part; int np; Bound bd; double* ws; };      // ws: the norms are written there (by one workgroup); may be null
__device__ __forceinline__ double factor(const Source& s) {
    if (s.bd.max_norm < 0.0) return 1.0;
    const Norms r = join_partials<THREADS>(s.part, s.np, s.bd);
    if (s.ws && blockIdx.x == 0 && threadIdx.x == 0) put_norms(r, s.ws);
    return r.c;
}

// y = c x (p[0] = x, p[1] = y).  A list inside the bound (c = 1) is left untouched in place.
template <bool NT>
__global__ __launch_bounds__(THREADS) void clip_kernel(const Table<2> t, const Source s) {
    const double c = factor(s);
    chunks<2, true>(t, [&](double* const* p, long long a, long long n) {
        if (c == 1.0 && p[0] == p[1]) return;
        d2 v[UNROLL];
        load_chunk<false>(v, p[0], a, n);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) v[u] *= c;
        store_chunk<NT>(v, p[1], a, n);
    });
}

struct Step { double lr, mu, one_minus_tau; int first; };

// d = c g -> the new momentum (MOMENTUM), p -> the new parameters
template <bool MOMENTUM> __device__ __forceinline__ void step_pair(d2& p, d2& d, d2 m, double c, const Step& s) {
    d *= c;
    if (MOMENTUM && !s.first) d = m * s.mu + d * s.one_minus_tau;
    p -= d * s.lr;
}

// p[0] = parameters, p[1] = gradients, p[2] = momentum buffers (MOMENTUM)
template <bool MOMENTUM, bool NT>
__global__ __launch_bounds__(THREADS) void sgd_kernel(const Table<MOMENTUM ? 3 : 2> t, const Step s, const Source src) {
    const double c = factor(src);
    chunks<MOMENTUM ? 3 : 2, true>(t, [&](double* const* p, long long a, long long n) {
        d2 x[UNROLL], d[UNROLL], m[UNROLL];
        load_chunk<false>(d, p[1], a, n);
        if (MOMENTUM && !s.first) load_chunk<false>(m, p[MOMENTUM ? 2 : 0], a, n);
        load_chunk<false>(x, p[0], a, n);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) step_pair<MOMENTUM>(x[u], d[u], m[u], c, s);
        if (MOMENTUM) store_chunk<NT>(d, p[MOMENTUM ? 2 : 0], a, n);
        store_chunk<NT>(x, p[0], a, n);
    });
}

// Short lists: one workgroup, one launch, the list in registers between the norm and its second use.  Its 16 waves take pieces of 128 doubles,
// ROUNDS of them each.
constexpr int PIECE = 128, SMALL_THREADS = 1024, SMALL_WAVES = SMALL_THREADS / 64;
enum { OP_NORMS, OP_CLIP, OP_SGD, OP_SGD_MOMENTUM };
template <int OP> struct Shape {
    static constexpr int NP = OP == OP_NORMS ? 1 : OP == OP_SGD_MOMENTUM ? 3 : 2, READ = OP >= OP_SGD ? 1 : 0, ROUNDS = OP == OP_NORMS ? 6 : 3;
};

__device__ __forceinline__ d2 load_piece(const double* x, int i, int n) {
    d2 v = {0.0, 0.0};
    if (i + 1 < n) v = load2<false>(x + i);
    else if (i < n) v.x = x[i];
    return v;
}
__device__ __forceinline__ void store_piece(d2 v, double* x, int i, int n) {
    if (i + 1 < n) store2<false>(x + i, v);
    else if (i < n) x[i] = v.x;
}

template <int OP, bool CPLX>
__global__ __launch_bounds__(SMALL_THREADS) void small_kernel(const Table<Shape<OP>::NP> t, const Bound bd, const Step s, double* ws) {
    using S = Shape<OP>;
    Finder<S::NP> at(t);
    const unsigned G = t.first[Table<S::NP>::N];
    const int lane = threadIdx.x & 63;
    const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    d2 v[S::ROUNDS], x[S::ROUNDS], m[S::ROUNDS];
#pragma unroll
    for (int r = 0; r < S::ROUNDS; ++r) {
        const unsigned q = wave + r * SMALL_WAVES;
        if (q < G) {
            at.find(q, PIECE);
            const int i = (int)(q - at.f) * PIECE + 2 * lane, n = (int)at.n;
            v[r] = load_piece(at.p[S::READ], i, n);
            if (OP >= OP_SGD) x[r] = load_piece(at.p[0], i, n);
            if (OP == OP_SGD_MOMENTUM) m[r] = load_piece(at.p[S::NP - 1], i, n);
        }
    }
    Acc acc;
#pragma unroll
    for (int r = 0; r < S::ROUNDS; ++r)
        if (wave + r * SMALL_WAVES < G) add<CPLX>(acc, v[r]);
    const Norms nr = finish(reduce_block<SMALL_WAVES>(part_of<CPLX>(acc)), bd);
    if (threadIdx.x == 0) put_norms(nr, ws);
    if (OP == OP_NORMS) return;
#pragma unroll
    for (int r = 0; r < S::ROUNDS; ++r) {
        const unsigned q = wave + r * SMALL_WAVES;
        if (q >= G) return;
        at.find(q, PIECE);
        const int i = (int)(q - at.f) * PIECE + 2 * lane, n = (int)at.n;
        if (OP == OP_CLIP) {
            if (nr.c != 1.0 || at.p[S::NP - 1] != at.p[0]) store_piece(v[r] * nr.c, at.p[S::NP - 1], i, n);
        } else {
            step_pair<OP == OP_SGD_MOMENTUM>(x[r], v[r], m[r], nr.c, s);
            if (OP == OP_SGD_MOMENTUM) store_piece(v[r], at.p[S::NP - 1], i, n);
            store_piece(x[r], at.p[0], i, n);
        }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------

// A list of nt tensors with NP pointers each
template <int NP> struct Lists {
    int nt; const double* const* p[NP]; const long long* n; long long unit;      // unit: doubles per element
};

int list_error(ctm_ctx* ctx, const char* name, const std::string& what) {
    ctx->set_error(std::string(name) + ": " + what);
    return CTM_ERR_BADARG;
}

int check_device(ctm_ctx* ctx, const char* name) {
    int dev = -1;
    CTM_HIP_CHECK(ctx, hipGetDevice(&dev));
    if (dev != ctx->device) return list_error(ctx, name, "the context belongs to device " + std::to_string(ctx->device) + ", device " + std::to_string(dev) + " is current");
    return CTM_OK;
}

// Lengths, pointers and the memory that is written: no written range may overlap any other range of the call (in a clip the range that is read
// and written under the same index may be one and the same).
template <int NP> int check_lists(ctm_ctx* ctx, const char* name, const Lists<NP>& L, const bool (&written)[NP], int same_as_first) {
    if (L.nt < 0) return list_error(ctx, name, "negative number of tensors");
    if (L.nt && !L.n) return list_error(ctx, name, "lengths missing");
    for (int j = 0; j < NP; ++j) if (L.nt && !L.p[j]) return list_error(ctx, name, "pointers missing");
    long long total = 0;
    bool any_written = false;
    for (int i = 0; i < L.nt; ++i) {
        if (L.n[i] < 0 || L.n[i] > (1LL << 40)) return list_error(ctx, name, "length of tensor " + std::to_string(i) + " out of range");
        total += L.n[i];
        if (total > (1LL << 40)) return list_error(ctx, name, "list too long");
        if (!L.n[i]) continue;
        for (int j = 0; j < NP; ++j) {
            if (!L.p[j][i]) return list_error(ctx, name, "null pointer for tensor " + std::to_string(i));
            if ((uintptr_t)L.p[j][i] % 8) return list_error(ctx, name, "tensor " + std::to_string(i) + " is not aligned to 8 bytes");
        }
    }
    for (int j = 0; j < NP; ++j) any_written |= written[j];
    if (!any_written) return CTM_OK;
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
        if (x.a < end_written || (x.w && x.a < end_any)) return list_error(ctx, name, "a tensor that is written overlaps another tensor of the call");
        if (x.b > end_any) end_any = x.b;
        if (x.w && x.b > end_written) end_written = x.b;
    }
    return CTM_OK;
}

// The next launch's table from tensor `i` on; returns the index behind its last tensor.
constexpr uintptr_t SPAN = (uintptr_t)8 << 32;           // what 32-bit counts of doubles reach
template <int NP> int fill(const Lists<NP>& L, int i, Table<NP>& t, int chunk = CHUNK) {
    constexpr int N = Table<NP>::N;
    int take[N], k = 0;
    uintptr_t lo[NP], hi[NP];
    for (; i < L.nt && k < N; ++i) {
        if (!L.n[i]) continue;
        bool fits = true;
        uintptr_t a[NP], b[NP];
        for (int j = 0; j < NP; ++j) {
            const uintptr_t x = (uintptr_t)L.p[j][i];
            a[j] = k && lo[j] < x ? lo[j] : x;
            b[j] = k && hi[j] > x ? hi[j] : x;
            fits &= b[j] - a[j] < SPAN;
        }
        if (!fits) break;                                // (never for the first tensor)
        for (int j = 0; j < NP; ++j) { lo[j] = a[j]; hi[j] = b[j]; }
        take[k++] = i;
    }
    unsigned q = 0;
    for (int j = 0; j < NP; ++j) t.base[j] = (double*)(k ? lo[j] : 0);
    for (int e = 0; e < k; ++e) {
        const long long n = L.n[take[e]] * L.unit, c = (n + chunk - 1) / chunk;
        for (int j = 0; j < NP; ++j) t.offset[j][e] = (unsigned)(((uintptr_t)L.p[j][take[e]] - lo[j]) / 8);
        t.first[e] = q;
        t.tail[e] = (unsigned short)(n - (c - 1) * chunk - 1);
        q += (unsigned)c;
    }
    for (int e = k; e <= N; ++e) t.first[e] = q;
    return i;
}

// launch on the caller's stream, CTM_LAUNCH's checks
#define GRADS_LAUNCH(ctx, stream, kernel, grid, block, ...)                                                       \
    do {                                                                                                          \
        if (g_ctm_sync_launch) ctm_note_launch(#kernel);                                                          \
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(block), 0, stream, __VA_ARGS__);                              \
        hipError_t _le = hipGetLastError();                                                                       \
        if (_le == hipSuccess && g_ctm_sync_launch) _le = hipStreamSynchronize(stream);                           \
        if (_le != hipSuccess) {                                                                                  \
            (ctx)->set_error(std::string("launch of " #kernel ": ") + hipGetErrorString(_le));                    \
            return CTM_ERR_HIP;                                                                                   \
        }                                                                                                         \
    } while (0)

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
template <int OP> bool small(ctm_ctx* ctx, hipStream_t s, const Lists<Shape<OP>::NP>& L, const Size& z, Bound bd, const Step& st, double* ws, int* status) {
    Table<Shape<OP>::NP> t;
    if (z.tensors > t.N || z.pieces > Shape<OP>::ROUNDS * SMALL_WAVES) return false;
    if (fill(L, 0, t, PIECE) < L.nt) return false;       // (tensors too far from each other)
    *status = [&]() -> int {
        if (ctx->cplx) GRADS_LAUNCH(ctx, s, (small_kernel<OP, true>), 1, SMALL_THREADS, t, bd, st, ws);
        else GRADS_LAUNCH(ctx, s, (small_kernel<OP, false>), 1, SMALL_THREADS, t, bd, st, ws);
        return CTM_OK;
    }();
    return true;
}

// Lists that do not fit the 256 MB last-level cache are read once without a claim on it (545 MB: 82 us against 87); stores of lists longer than
// the 32 MB of L2 cache bypass it (545 MB scaled in 185 us against 188 ... 229, 1.1 GB after its norm pass in 556 against 591).
constexpr long long LLC_BYTES = 256LL << 20, L2_BYTES = 32LL << 20;

template <bool NT> int partials(ctm_ctx* ctx, hipStream_t s, const Lists<1>& L, const Size& z, double* ws, int* np) {
    *np = 0;
    Part* part = (Part*)(ws + WS_HEAD);
    for (int i = 0; i < L.nt;) {
        Table<1> t;
        i = fill(L, i, t);
        const unsigned long long g = t.first[t.N];
        if (!g) break;
        unsigned long long grid = z.chunks <= PARTIALS ? g : PARTIALS * g / z.chunks;
        if (grid < 1) grid = 1;
        if (ctx->cplx) GRADS_LAUNCH(ctx, s, (norm_partials_kernel<true, NT>), (unsigned)grid, THREADS, t, part + *np);
        else GRADS_LAUNCH(ctx, s, (norm_partials_kernel<false, NT>), (unsigned)grid, THREADS, t, part + *np);
        *np += (int)grid;
    }
    return CTM_OK;
}

int norm_pass(ctm_ctx* ctx, hipStream_t s, const Lists<1>& L, const Size& z, double* ws, int* np) {
    return z.bytes > LLC_BYTES ? partials<true>(ctx, s, L, z, ws, np) : partials<false>(ctx, s, L, z, ws, np);
}

// Second pass over a list: launch(table, grid, source) for every table of it.
constexpr unsigned MAX_GRID = 8192;
template <int NP, class F> int second_pass(const Lists<NP>& L, Source src, F&& launch) {
    for (int i = 0; i < L.nt;) {
        Table<NP> t;
        i = fill(L, i, t);
        const unsigned g = t.first[t.N];
        if (!g) break;
        CTM_TRY(launch(t, g < MAX_GRID ? g : MAX_GRID, src));
        src.ws = nullptr;                    // the norms are written once
    }
    return CTM_OK;
}

template <bool MOMENTUM> int sgd(ctm_ctx* ctx, hipStream_t s, const Lists<MOMENTUM ? 3 : 2>& L, const Size& z, const Step& st, const Source& src) {
    return second_pass(L, src, [&](const Table<MOMENTUM ? 3 : 2>& t, unsigned grid, const Source& f) -> int {
        if (z.bytes > L2_BYTES) GRADS_LAUNCH(ctx, s, (sgd_kernel<MOMENTUM, true>), grid, THREADS, t, st, f);
        else GRADS_LAUNCH(ctx, s, (sgd_kernel<MOMENTUM, false>), grid, THREADS, t, st, f);
        return CTM_OK;
    });
}

}  // namespace

extern "C" {

int ctm_grad_norms(ctm_ctx* ctx, void* hip_stream, int nt, const double* const* x, const long long* n, double* ws, long long ws_doubles) {
    return ctm_entry(ctx, "ctm_grad_norms", [&]() -> int {
    CTM_TRY(check_device(ctx, "grad_norms"));
    const bool written[1] = {false};
    CTM_TRY(check_lists<1>(ctx, "grad_norms", Lists<1>{nt, {x}, n, ctx->cplx ? 2 : 1}, written, 0));
    if (!ws || ws_doubles < CTM_GRAD_WS_DOUBLES((long long)nt)) return list_error(ctx, "grad_norms", "workspace too small (CTM_GRAD_WS_DOUBLES)");
    hipStream_t s = (hipStream_t)hip_stream;
    const Lists<1> L{nt, {x}, n, ctx->cplx ? 2 : 1};
    const Size z = size_of(n, nt, L.unit);
    const Bound none{-1.0, 0};
    int status, np;
    if (small<OP_NORMS>(ctx, s, L, z, none, Step{}, ws, &status)) return status;
    CTM_TRY(norm_pass(ctx, s, L, z, ws, &np));
    GRADS_LAUNCH(ctx, s, norm_finish_kernel, 1, 1024, (const Part*)(ws + WS_HEAD), np, none, ws);
    return CTM_OK;
    });
}

int ctm_grad_clip(ctm_ctx* ctx, void* hip_stream, int nt, const double* const* x, double* const* y, const long long* n, int norm_type,
                  double max_norm, double* ws, long long ws_doubles) {
    return ctm_entry(ctx, "ctm_grad_clip", [&]() -> int {
    CTM_TRY(check_device(ctx, "grad_clip"));
    const bool written[2] = {false, true};
    Lists<2> L{nt, {x, (const double* const*)y}, n, ctx->cplx ? 2 : 1};
    CTM_TRY(check_lists<2>(ctx, "grad_clip", L, written, 1));
    if (!(max_norm >= 0.0)) return list_error(ctx, "grad_clip", "max_norm must be >= 0");
    if (norm_type != CTM_NORM_2 && norm_type != CTM_NORM_INF) return list_error(ctx, "grad_clip", "norm_type must be CTM_NORM_2 or CTM_NORM_INF");
    if (!ws || ws_doubles < CTM_GRAD_WS_DOUBLES((long long)nt)) return list_error(ctx, "grad_clip", "workspace too small (CTM_GRAD_WS_DOUBLES)");
    hipStream_t s = (hipStream_t)hip_stream;
    const Bound bd{max_norm, norm_type == CTM_NORM_INF};
    const Size z = size_of(n, nt, L.unit);
    int status, np;
    if (small<OP_CLIP>(ctx, s, L, z, bd, Step{}, ws, &status)) return status;
    CTM_TRY(norm_pass(ctx, s, Lists<1>{nt, {x}, n, L.unit}, z, ws, &np));
    return second_pass(L, Source{(const Part*)(ws + WS_HEAD), np, bd, ws}, [&](const Table<2>& t, unsigned grid, const Source& f) -> int {
        if (z.bytes > L2_BYTES) GRADS_LAUNCH(ctx, s, clip_kernel<true>, grid, THREADS, t, f);
        else GRADS_LAUNCH(ctx, s, clip_kernel<false>, grid, THREADS, t, f);
        return CTM_OK;
    });
    });
}

int ctm_sgd_step(ctm_ctx* ctx, void* hip_stream, int nt, double* const* p, const double* const* g, double* const* m, const long long* n,
                 double lr, double momentum, double dampening, int first, int norm_type, double max_norm, double* ws, long long ws_doubles) {
    return ctm_entry(ctx, "ctm_sgd_step", [&]() -> int {
    CTM_TRY(check_device(ctx, "sgd_step"));
    Lists<3> L3{nt, {(const double* const*)p, g, (const double* const*)m}, n, ctx->cplx ? 2 : 1};
    Lists<2> L2{nt, {(const double* const*)p, g}, n, ctx->cplx ? 2 : 1};
    if (m) { const bool w[3] = {true, false, true}; CTM_TRY(check_lists<3>(ctx, "sgd_step", L3, w, 0)); }
    else { const bool w[2] = {true, false}; CTM_TRY(check_lists<2>(ctx, "sgd_step", L2, w, 0)); }
    if (nt > 0 && !m && momentum != 0.0) return list_error(ctx, "sgd_step", "momentum needs the momentum buffers");
    hipStream_t s = (hipStream_t)hip_stream;
    const bool bounded = max_norm >= 0.0;
    if (max_norm != max_norm) return list_error(ctx, "sgd_step", "max_norm is NaN");
    if (bounded) {
        if (norm_type != CTM_NORM_2 && norm_type != CTM_NORM_INF) return list_error(ctx, "sgd_step", "norm_type must be CTM_NORM_2 or CTM_NORM_INF");
        if (!ws || ws_doubles < CTM_GRAD_WS_DOUBLES((long long)nt)) return list_error(ctx, "sgd_step", "workspace too small (CTM_GRAD_WS_DOUBLES)");
    }
    const Step st{lr, momentum, 1.0 - dampening, first};
    const Size z = size_of(n, nt, L2.unit);
    Source src{nullptr, 0, Bound{bounded ? max_norm : -1.0, norm_type == CTM_NORM_INF}, ws};
    if (bounded) {
        int status;
        if (m ? small<OP_SGD_MOMENTUM>(ctx, s, L3, z, src.bd, st, ws, &status) : small<OP_SGD>(ctx, s, L2, z, src.bd, st, ws, &status)) return status;
        CTM_TRY(norm_pass(ctx, s, Lists<1>{nt, {g}, n, L2.unit}, z, ws, &src.np));
        src.part = (const Part*)(ws + WS_HEAD);
    }
    return m ? sgd<true>(ctx, s, L3, z, st, src) : sgd<false>(ctx, s, L2, z, st, src);
    });
}

}  // extern "C"
