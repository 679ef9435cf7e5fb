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

// Tensors of one launch: their table travels by value in the kernel arguments (no host-to-device copy, so a call may be captured).  64 = one
// wave: the lookup "which tensor holds granule q" is one comparison per lane and a population count.
constexpr int TAB = 64;
constexpr int GRANULE = 1024;          // doubles: unit in which the work of a launch is dealt out to its workgroups
constexpr int THREADS = 256;
constexpr int WS_HEAD = 4;             // ws: N2, Ninf, c, unused, then the partial results (4 doubles each)
constexpr int PARTIALS = 1024;         // workgroups of the norm pass over all launches, up to one more per launch

template <int NP> struct Table {
    double* p[NP][TAB];
    long long n[TAB];                  // doubles (a complex element counts two)
    unsigned first[TAB + 1];           // granules before tensor t; entries behind the last tensor hold the total
};

typedef double d2 __attribute__((ext_vector_type(2)));
typedef d2 d2u __attribute__((aligned(8)));          // 16-byte access at 8-byte alignment: views into a flat buffer start anywhere

// tensor of granule q: the lanes of a wave compare one table entry each
template <int NP> __device__ __forceinline__ int tensor_of(const Table<NP>& t, unsigned q) {
    const int lane = threadIdx.x & 63;
    return __popcll(__ballot(t.first[lane + 1] <= q));
}

// Runs body(tensor, begin, end) over the segments (in doubles) of this workgroup's share of the granules.
template <int NP, class F> __device__ __forceinline__ void segments(const Table<NP>& t, F&& body) {
    const unsigned long long G = t.first[TAB];
    unsigned q = (unsigned)(G * blockIdx.x / gridDim.x);
    const unsigned qe = (unsigned)(G * (blockIdx.x + 1) / gridDim.x);
    while (q < qe) {
        const int k = __builtin_amdgcn_readfirstlane(tensor_of(t, q));
        const unsigned f = t.first[k], l = t.first[k + 1];
        const unsigned e = l < qe ? l : qe;
        const long long n = t.n[k];
        const long long a = (long long)(q - f) * GRANULE, b = (long long)(e - f) * GRANULE;
        body(k, a, b < n ? b : n);
        q = e;
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

// Partial result of a workgroup of `WAVES` waves, valid on thread 0.
template <int WAVES> __device__ __forceinline__ Part reduce_block(Part p) {
    __shared__ Part sh[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    p.med = wave_sum(p.med);
    if (__any(p.big != 0.0)) p.big = wave_sum(p.big);          // (true for NaN)
    if (__any(p.small != 0.0)) p.small = wave_sum(p.small);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) p.top = umax(p.top, __shfl_xor(p.top, o));
    if (WAVES == 1) return p;
    if (lane == 0) sh[wave] = p;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < WAVES; ++w) {
            p.big += sh[w].big; p.med += sh[w].med; p.small += sh[w].small; p.top = umax(p.top, sh[w].top);
        }
    return p;
}

template <bool CPLX> __device__ __forceinline__ Part part_of(const Acc& a) {
    Part p{a.big, a.med, a.small, a.top};
    if (CPLX) p.top = umax(bits(sqrt(__longlong_as_double((long long)a.top))), a.top_far);
    return p;
}

struct Bound { double max_norm; int inf_norm; };      // max_norm < 0: no bound

// N2, Ninf and the factor c from the three range sums
__device__ __forceinline__ void finish(const Part& p, Bound bd, double* ws) {
    double n2;
    if (p.big != 0.0) n2 = sqrt(fma(p.med * 0x1p-600, 0x1p-600, p.big)) * 0x1p600;
    else if (p.med != 0.0) n2 = sqrt(fma(p.small * 0x1p-600, 0x1p-600, p.med));
    else n2 = sqrt(p.small) * 0x1p-600;
    const double ninf = __longlong_as_double((long long)p.top);
    const double n = bd.inf_norm ? ninf : n2;
    ws[0] = n2;
    ws[1] = ninf;
    ws[2] = (bd.max_norm < 0.0 || n <= bd.max_norm) ? 1.0 : bd.max_norm / n;      // NaN norm: NaN
}

template <bool CPLX>
__global__ __launch_bounds__(THREADS) void norm_partials_kernel(const Table<1> t, Part* out) {
    Acc acc;
    segments(t, [&](int k, long long a, long long b) {
        const double* x = t.p[0][k];
        long long i = a + 2 * threadIdx.x;
        for (; i + 3 * 2 * THREADS + 1 < b; i += 4 * 2 * THREADS) {
            d2 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = *(const d2u*)(x + i + u * 2 * THREADS);
#pragma unroll
            for (int u = 0; u < 4; ++u) add<CPLX>(acc, v[u]);
        }
        for (; i + 1 < b; i += 2 * THREADS) add<CPLX>(acc, *(const d2u*)(x + i));
        if (i < b) { d2 v = {x[i], 0.0}; add<CPLX>(acc, v); }          // (real tensors of odd length)
    });
    const Part p = reduce_block<THREADS / 64>(part_of<CPLX>(acc));
    if (threadIdx.x == 0) out[blockIdx.x] = p;
}

__global__ __launch_bounds__(1024) void norm_finish_kernel(const Part* part, int np, Bound bd, double* ws) {
    Part p{0.0, 0.0, 0.0, 0};
    for (int i = threadIdx.x; i < np; i += 1024) {
        const Part q = part[i];
        p.big += q.big; p.med += q.med; p.small += q.small; p.top = umax(p.top, q.top);
    }
    p = reduce_block<16>(p);
    if (threadIdx.x == 0) finish(p, bd, ws);
}

// y = c x (p[0] = x, p[1] = y).  A list inside the bound (c = 1) is left untouched in place.
__global__ __launch_bounds__(THREADS) void clip_kernel(const Table<2> t, const double* ws) {
    const double c = ws[2];
    segments(t, [&](int k, long long a, long long b) {
        const double* x = t.p[0][k];
        double* y = t.p[1][k];
        if (c == 1.0 && x == y) return;
        for (long long i = a + 2 * threadIdx.x; i < b; i += 2 * THREADS) {
            if (i + 1 < b) { const d2 v = *(const d2u*)(x + i); *(d2u*)(y + i) = v * c; }
            else y[i] = x[i] * c;
        }
    });
}

struct Step { double lr, mu, one_minus_tau; int first, bounded; };

// p[0] = parameters, p[1] = gradients, p[2] = momentum buffers (MOMENTUM)
template <bool MOMENTUM, class V> __device__ __forceinline__ void step_one(double* p, const double* g, double* m, long long i, double c, const Step& s) {
    V d = *(const V*)(g + i) * c;
    if (MOMENTUM) {
        if (!s.first) d = *(const V*)(m + i) * s.mu + d * s.one_minus_tau;
        *(V*)(m + i) = d;
    }
    *(V*)(p + i) = *(const V*)(p + i) - d * s.lr;
}

template <bool MOMENTUM>
__global__ __launch_bounds__(THREADS) void sgd_kernel(const Table<MOMENTUM ? 3 : 2> t, Step s, const double* ws) {
    const double c = s.bounded ? ws[2] : 1.0;
    segments(t, [&](int k, long long a, long long b) {
        double* p = t.p[0][k];
        const double* g = t.p[1][k];
        double* m = MOMENTUM ? t.p[MOMENTUM ? 2 : 0][k] : nullptr;
        for (long long i = a + 2 * threadIdx.x; i < b; i += 2 * THREADS) {
            if (i + 1 < b) step_one<MOMENTUM, d2u>(p, g, m, i, c, s);
            else step_one<MOMENTUM, double>(p, g, m, i, c, s);
        }
    });
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------

// A list of nt tensors with NP pointers each, cut into launches of at most TAB non-empty tensors.
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
template <int NP> int fill(const Lists<NP>& L, int i, Table<NP>& t) {
    int k = 0;
    unsigned q = 0;
    for (; i < L.nt && k < TAB; ++i) {
        if (!L.n[i]) continue;
        for (int j = 0; j < NP; ++j) t.p[j][k] = const_cast<double*>(L.p[j][i]);
        t.n[k] = L.n[i] * L.unit;
        t.first[k++] = q;
        q += (unsigned)((t.n[k - 1] + GRANULE - 1) / GRANULE);
    }
    for (int j = k; j <= TAB; ++j) t.first[j] = q;
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

unsigned granules_of(const long long* n, int nt, long long unit) {
    unsigned long long g = 0;
    for (int i = 0; i < nt; ++i) g += (unsigned long long)((n[i] * unit + GRANULE - 1) / GRANULE);
    return (unsigned)g;
}

int norms(ctm_ctx* ctx, hipStream_t s, int nt, const double* const* x, const long long* n, Bound bd, double* ws) {
    Lists<1> L{nt, {x}, n, ctx->cplx ? 2 : 1};
    const unsigned long long total = granules_of(n, nt, L.unit);
    Part* part = (Part*)(ws + WS_HEAD);
    int np = 0;
    for (int i = 0; i < nt;) {
        Table<1> t;
        i = fill(L, i, t);
        const unsigned long long g = t.first[TAB];
        if (!g) break;
        unsigned long long grid = PARTIALS * g / total;
        grid = grid < 1 ? 1 : grid > g ? g : grid;
        if (ctx->cplx) GRADS_LAUNCH(ctx, s, norm_partials_kernel<true>, (unsigned)grid, THREADS, t, part + np);
        else GRADS_LAUNCH(ctx, s, norm_partials_kernel<false>, (unsigned)grid, THREADS, t, part + np);
        np += (int)grid;
    }
    GRADS_LAUNCH(ctx, s, norm_finish_kernel, 1, 1024, (const Part*)part, np, bd, ws);
    return CTM_OK;
}

constexpr unsigned MAX_GRID = 4096;

}  // namespace

extern "C" {

int ctm_grad_norms(ctm_ctx* ctx, void* hip_stream, int nt, const double* const* x, const long long* n, double* ws, long long ws_doubles) {
    return ctm_entry(ctx, "ctm_grad_norms", [&]() -> int {
    CTM_TRY(check_device(ctx, "grad_norms"));
    const bool written[1] = {false};
    CTM_TRY(check_lists<1>(ctx, "grad_norms", Lists<1>{nt, {x}, n, ctx->cplx ? 2 : 1}, written, 0));
    if (!ws || ws_doubles < CTM_GRAD_WS_DOUBLES((long long)nt)) return list_error(ctx, "grad_norms", "workspace too small (CTM_GRAD_WS_DOUBLES)");
    return norms(ctx, (hipStream_t)hip_stream, nt, x, n, Bound{-1.0, 0}, ws);
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
    CTM_TRY(norms(ctx, s, nt, x, n, Bound{max_norm, norm_type == CTM_NORM_INF}, ws));
    for (int i = 0; i < nt;) {
        Table<2> t;
        i = fill(L, i, t);
        const unsigned g = t.first[TAB];
        if (!g) break;
        GRADS_LAUNCH(ctx, s, clip_kernel, g < MAX_GRID ? g : MAX_GRID, THREADS, t, (const double*)ws);
    }
    return CTM_OK;
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
        CTM_TRY(norms(ctx, s, nt, g, n, Bound{max_norm, norm_type == CTM_NORM_INF}, ws));
    }
    const Step st{lr, momentum, 1.0 - dampening, first, bounded};
    for (int i = 0; i < nt;) {
        unsigned q;
        if (m) {
            Table<3> t;
            i = fill(L3, i, t);
            if (!(q = t.first[TAB])) break;
            GRADS_LAUNCH(ctx, s, sgd_kernel<true>, q < MAX_GRID ? q : MAX_GRID, THREADS, t, st, (const double*)ws);
        } else {
            Table<2> t;
            i = fill(L2, i, t);
            if (!(q = t.first[TAB])) break;
            GRADS_LAUNCH(ctx, s, sgd_kernel<false>, q < MAX_GRID ? q : MAX_GRID, THREADS, t, st, (const double*)ws);
        }
    }
    return CTM_OK;
    });
}

}  // extern "C"
