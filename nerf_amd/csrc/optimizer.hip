// The work between a backward pass and the next forward pass, over a list of tensors: the global norm of the
// gradients, clipping by it, and the AdamW step that clips while it reads the gradients.
//
//   norm      N = (sum_i sum_j |g_ij|^p)^(1/p) for p = 1, 2, or max_ij |g_ij|
//   clip      g <- c g,  c = min(1, max_norm / (N + 1e-6))
//   AdamW     g' = c g,  m <- b1 m + (1 - b1) g',  v <- b2 v + (1 - b2) g'^2,  t <- t + 1
//             w <- w - lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + wd w)
//
// All of it is bound by memory.  The tensors of a list reach a kernel by value, as a table in its arguments (no copy
// to the device, nothing that a captured graph would have to keep alive); a list longer than a table goes out as
// several launches.  Each tensor is cut into chunks, which the workgroups of a launch take in turn, so that all of them
// together sweep through memory.  The norm is one launch that leaves a partial sum per workgroup in the caller's
// workspace; every workgroup of the launch that needs the norm adds those up for itself, in one fixed order, so that
// there are no atomics, no waiting between workgroups and no launch in between.  The order of a sum goes by the list and
// by where its tensors start within a line of memory: alike in these, two calls give the same bits.
#include <stdlib.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"

namespace {

constexpr int kThreads = 256;

// How a kernel's launches are cut: at most `groups` workgroups, and chunks of `least` elements (one access per lane) while
// the list is short, so that every compute unit gets some, up to `most` for a long one.  What the workgroups touch at one
// time (groups x chunk, in each of the tensors' arrays) is kept to a few megabytes: AdamW over 1e8 fp32 parameters in 128
// tensors takes 618 us with 2048 workgroups and chunks of 16384, 578 with 1024 and 4096, 530 with 768 and 2048, 524 with
// 512 and 2048 (551 with 512 and 4096, 536 with 512 and 1024, 580 with 640 and 2048, 608 with 256 and 2048); the norm of
// 4.3 GB 628 us with 2048 and 16384, 616 with 2048 and 8192, 611 with 1024 and 4096 to 16384, 593 with 512 and 8192 (120 MB
// 20.9 instead of 19.9).  Its inner loop wants four accesses per lane and chunk: with two 758 us, and 5e8 bf16 elements
// 189 us instead of 147.
struct Cut {
    int groups, least, most;
};
constexpr int kNormGroups = 1024;
constexpr Cut norm_cut(int size) { return {kNormGroups, 4096 / size, 32768 / size}; }
constexpr Cut scale_cut(int size) { return {1024, 4096 / size, 16384 / size}; }
constexpr Cut adam_cut(int) { return {512, 1024, 2048}; }

// Accesses past the caches (non-temporal ones), in bytes of what a call reads and writes.  A norm that nothing follows:
// 4.3 GB 611 us against 690 through the caches, 120 MB 19.9 against 21.3 and 40 MB 11 either way; 120 MB that were
// written just before 58.3 against 55.2 (with the writing).  An update with its norm: AdamW of 140 MB 33.8 against 31.8, of
// 280 MB 58.1 against 54.6, of 2.8 GB 524 against 633, of 5.6 GB 1101 against 1246.  The norm ahead of an update stays
// in the caches at any size: even where they hold only part of the gradients the update finds some there (AdamW of
// 2.8 GB 524 us against 559, of 5.6 GB 1101 against 1126).
constexpr int64_t kMiB = 1 << 20;
constexpr int64_t kNormStream = 64 * kMiB;
constexpr int64_t kUpdateStream = 192 * kMiB;

// The tables stay below 4 KB of kernel arguments.  A tensor's chunks are counted from the start of the line of memory that
// holds its first element (`shift` elements before it), so that a wave's accesses cover whole lines but at the two ends:
// AdamW of 3e7 bf16 parameters that start at odd places 184 us, 205 with accesses that are aligned to 16 bytes only, 182
// where each starts on a line.
template <int CAP>
struct Chunks {
    static constexpr int kCap = CAP;
    int end[CAP];           // chunks of the tensors up to and including this one
    int tail[CAP];          // elements of its last chunk (with `shift` where that is its first one too)
    int n, chunk;
};

struct ListTable : Chunks<224> {
    void* ptr[kCap];
};

struct NormStepTable : Chunks<120> {    // with the step counters, which the norm's launch copies to the workspace
    void* ptr[kCap];
    const float* step[kCap];
    int id[kCap];           // place in the caller's list
};

struct AdamTable : Chunks<56> {
    void* p[kCap];
    const void* g[kCap];
    float* m[kCap];
    float* v[kCap];
    float* w[kCap];         // 32-bit master weights (16-bit parameters)
    float* step[kCap];
    int id[kCap];
};

constexpr int kStepCap = 256;
struct StepTable {
    const float* step[kStepCap];
    int n, first_tensor;
};

struct Clip {
    const double* partials;         // null: no norm is taken
    int n_partials, kind, skip_nonfinite;
    double max_norm;
    float* norm;                    // nullable
};

struct AdamArgs {
    const float* lr_ptr;            // null: lr
    float lr, beta1, beta2, eps, decay, rest1, rest2;       // rest = 1 - beta, rounded from 64 bits
    double ln1, ln2;                // ln(beta)
};

// Elements between the start of a pointer's line of memory and the pointer.
constexpr int kLine = 128;
__host__ __device__ inline int shift_of(const void* p, int size) { return (int)((uintptr_t)p % kLine) / size; }

// The workgroup's place in a table: chunk b as the stretch [lo, hi) of tensor t; lo is -shift in a tensor's first chunk.
// Among tensors of under a thousand chunks a workgroup's next chunk is mostly another tensor's, so that lookups are on
// the path of every chunk: the lanes of each wave hold the table's `end` in registers and compare all of it at once.
template <int CAP>
struct Cursor {
    static constexpr int kRegs = (CAP + 63) / 64;
    int ends[kRegs];
    int t = 0, first = 0, end = 0;      // the tensor, its first chunk and the first one behind it
    int shift = 0;
    int64_t numel = 0, lo = 0, hi = 0;

    __device__ __forceinline__ explicit Cursor(const Chunks<CAP>& tab) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < kRegs; ++k) ends[k] = 64 * k + lane < tab.n ? tab.end[64 * k + lane] : 0x7fffffff;
    }
    // The tensor of chunk b (b ascends) -> whether it is another one than before.
    __device__ __forceinline__ bool seek(const Chunks<CAP>& tab, int b) {
        if (b < end) return false;
        t = 0;
#pragma unroll
        for (int k = 0; k < kRegs; ++k) t += __popcll(__ballot(ends[k] <= b));
        first = t ? tab.end[t - 1] : 0;
        end = tab.end[t];
        return true;
    }
    // `lead`: the pointer whose lines the chunks go by.
    template <typename T>
    __device__ __forceinline__ void align(const Chunks<CAP>& tab, const T* lead) {
        shift = shift_of(lead, sizeof(T));
        numel = (int64_t)(end - first - 1) * tab.chunk + tab.tail[t] - shift;
    }
    __device__ __forceinline__ void range(const Chunks<CAP>& tab, int b) {
        lo = (int64_t)(b - first) * tab.chunk - shift;
        hi = lo + tab.chunk < numel ? lo + tab.chunk : numel;
    }
};

// One access of a lane.  The type promises no more alignment than an element's (the tensors of one parameter may lie at
// different places of their 16 bytes); the hardware takes such addresses in one access all the same, if more slowly.
// STREAM: past the caches, for lists that do not fit there.
template <typename T, int N, bool STREAM>
struct Pack {
    typedef T type __attribute__((ext_vector_type(N)));
    typedef type loose __attribute__((aligned(sizeof(T))));
    static __device__ __forceinline__ type load(const T* p) {
        return STREAM ? __builtin_nontemporal_load((const loose*)p) : *(const loose*)p;
    }
    static __device__ __forceinline__ void store(T* p, type x) {
        if (STREAM) __builtin_nontemporal_store(x, (loose*)p);
        else *(loose*)p = x;
    }
};

// ---- sums in a fixed order --------------------------------------------------------------------------------------
// Sums are held in 64 bits: the square of a 32-bit value is exact there, and neither overflows nor underflows, so the
// norm needs no scaling pass.  Maxima compare the bits of the absolute value, under which a NaN is the largest.

template <int KIND>
__device__ __forceinline__ double join(double a, double b) {
    if (KIND != NERF_NORM_MAX) return a + b;
    return __double_as_longlong(a) > __double_as_longlong(b) ? a : b;
}

template <int KIND>
__device__ __forceinline__ double take(double acc, float x) {
    if (KIND == NERF_NORM_L2) return fma((double)x, (double)x, acc);
    return join<KIND>(acc, (double)fabsf(x));
}

template <int KIND>
__device__ __forceinline__ double group_join(double x) {
    __shared__ double s[kThreads / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = join<KIND>(x, __shfl_xor(x, o));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    x = s[0];
#pragma unroll
    for (int i = 1; i < kThreads / 64; ++i) x = join<KIND>(x, s[i]);
    return x;
}

template <int KIND>
__device__ __forceinline__ double norm_of(const double* partials, int n) {
    constexpr int kDeep = 8;        // loads under way at once: every workgroup of the update waits for these
    double x = 0.0;
    for (int i = threadIdx.x; i < n; i += kDeep * kThreads) {
        double y[kDeep];
#pragma unroll
        for (int k = 0; k < kDeep; ++k) y[k] = i + k * kThreads < n ? partials[i + k * kThreads] : 0.0;
#pragma unroll
        for (int k = 0; k < kDeep; ++k) x = join<KIND>(x, y[k]);
    }
    x = group_join<KIND>(x);
    return KIND == NERF_NORM_L2 ? sqrt(x) : x;
}

__device__ __forceinline__ double norm_of(const Clip& c) {
    if (c.kind == NERF_NORM_L2) return norm_of<NERF_NORM_L2>(c.partials, c.n_partials);
    if (c.kind == NERF_NORM_L1) return norm_of<NERF_NORM_L1>(c.partials, c.n_partials);
    return norm_of<NERF_NORM_MAX>(c.partials, c.n_partials);
}

// factor * 2^exponent: formed in 64 bits, the factor rounded once to the 32 bits that the entries are multiplied in.  The
// exponent is 0 but for a coefficient below fp32's normal range, which would keep few bits there, or none: the entries
// that bring such a norm about are so large that their products are ordinary numbers again.
struct Scale {
    float factor = 1.f;
    int exponent = 0;
};

__device__ __forceinline__ Scale coefficient(double norm, double max_norm) {
    Scale s;
    const double d = norm + 1e-6;
    if (d <= max_norm) return s;
    double c = max_norm / d;                                // (a NaN norm gives NaN)
    if (c > 0.0 && c < 0x1p-126) c = frexp(c, &s.exponent);
    s.factor = (float)c;
    return s;
}

// One product in 32 bits; the power of two is exact, but for results below the normal range, and one instruction.
__device__ __forceinline__ float scaled(float x, const Scale& s) { return ldexpf(x * s.factor, s.exponent); }

// Bound by reading: 4.3 GB fp32 in one tensor 612 us, 7.0 TB/s; 6e8 bytes of bf16 in 389 tensors 107 us (two launches),
// 5.6 TB/s.  The 64-bit multiply-adds (one per element, half the fp32 rate) are a tenth of that.
template <typename T, int KIND, bool STREAM, typename Table>
__global__ __launch_bounds__(kThreads) void norm_partials(Table tab, double* partials, float* steps) {
    constexpr int V = 16 / sizeof(T), kStep = kThreads * V, kDeep = 4;
    using P = Pack<T, V, STREAM>;
    double acc[2] = {0.0, 0.0};
    const int total = tab.end[tab.n - 1];
    Cursor<Table::kCap> c(tab);
    const T* g = nullptr;
    for (int b = blockIdx.x; b < total; b += gridDim.x) {
        if (c.seek(tab, b)) {
            g = (const T*)tab.ptr[c.t];
            c.align(tab, g);
        }
        if constexpr (std::is_same<Table, NormStepTable>::value)
            if (b == c.first && threadIdx.x == 0) steps[tab.id[c.t]] = *tab.step[c.t];
        c.range(tab, b);
        int64_t i = c.lo + threadIdx.x * V;
        if (i < 0) {                                    // the first lanes of a tensor that starts inside a line
            for (int64_t j = 0; j < i + V && j < c.hi; ++j) acc[0] = take<KIND>(acc[0], (float)g[j]);
            i += kStep;
        }
        for (; i + (kDeep - 1) * kStep + V <= c.hi; i += kDeep * kStep) {
            typename P::type x[kDeep];
#pragma unroll
            for (int k = 0; k < kDeep; ++k) x[k] = P::load(g + i + k * kStep);
#pragma unroll
            for (int k = 0; k < kDeep; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j & 1] = take<KIND>(acc[j & 1], (float)x[k][j]);
        }
        for (; i + V <= c.hi; i += kStep) {
            const typename P::type x = P::load(g + i);
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j & 1] = take<KIND>(acc[j & 1], (float)x[j]);
        }
        for (; i < c.hi; ++i) acc[0] = take<KIND>(acc[0], (float)g[i]);     // the last lane's rest
    }
    const double sum = group_join<KIND>(join<KIND>(acc[0], acc[1]));
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kThreads) void norm_finish(Clip clip) {
    const double n = norm_of(clip);
    if (threadIdx.x == 0) *clip.norm = (float)n;
}

__global__ __launch_bounds__(kThreads) void read_steps(StepTable tab, float* steps) {
    const int i = threadIdx.x;
    if (i < tab.n) steps[tab.first_tensor + i] = *tab.step[i];
}

// Bound by memory; the product is a 32-bit one whatever the type, rounded to it once.  2 GB fp32 in 97 tensors: 655 us
// for 4 GB moved, 6.1 TB/s, behind a norm of 325.
template <typename T, bool STREAM>
__global__ __launch_bounds__(kThreads) void scale_by_norm(ListTable tab, Clip clip) {
    constexpr int V = 16 / sizeof(T), kStep = kThreads * V;
    using P = Pack<T, V, STREAM>;
    const double norm = norm_of(clip);
    if (blockIdx.x == 0 && threadIdx.x == 0) *clip.norm = (float)norm;
    const Scale s = coefficient(norm, clip.max_norm);
    const int total = tab.end[tab.n - 1];
    Cursor<ListTable::kCap> c(tab);
    T* g = nullptr;
    for (int b = blockIdx.x; b < total; b += gridDim.x) {
        if (c.seek(tab, b)) {
            g = (T*)tab.ptr[c.t];
            c.align(tab, g);
        }
        c.range(tab, b);
        for (int64_t i = c.lo + threadIdx.x * V; i < c.hi; i += kStep) {
            if (i >= 0 && i + V <= c.hi) {
                typename P::type x = P::load(g + i);
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] = (T)scaled((float)x[j], s);
                P::store(g + i, x);
            } else {
                for (int64_t j = i < 0 ? 0 : i; j < i + V && j < c.hi; ++j) g[j] = (T)scaled((float)g[j], s);
            }
        }
    }
}

__device__ __forceinline__ float of_lane(float x, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

struct Factors {
    Scale clip;
    float lr, inv1, inv2;           // inv1 = 1 / (1 - beta1^t), inv2 = 1 / sqrt(1 - beta2^t)
};

// One entry: its weight in 32 bits (the parameter itself, or its master), gradient and moments.
__device__ __forceinline__ void adamw_entry(float& w, float g, float& m, float& v, const AdamArgs& a, const Factors& f) {
    g = scaled(g, f.clip);
    m = a.beta1 * m + a.rest1 * g;
    v = a.beta2 * v + a.rest2 * (g * g);
    w -= f.lr * (m * f.inv1 / (sqrtf(v) * f.inv2 + a.eps) + a.decay * w);
}

// The weight that a step starts from.  The master stands for the parameter as long as it rounds to it: a parameter that
// was written from outside (a loaded checkpoint) is taken as it is.
template <typename T>
__device__ __forceinline__ float weight_of(T p, float master) {
    return (T)master == p ? master : (float)p;
}

// A 16-bit parameter is the rounding of its 32-bit master.  Left to itself the compiler forms the last multiply-add
// and the conversion to fp16 as one instruction, which rounds the exact sum once and so may end on the other neighbour
// than the rounding of the rounded sum: the value has to exist in 32 bits first.
__device__ __forceinline__ void keep_rounded(float& x) { asm("" : "+v"(x)); }

// Bound by memory: 28 bytes per fp32 parameter and 30 per 16-bit one; 1e8 fp32 parameters in 128 tensors 529 us with the
// norm, 3.2 GB at 6.0 TB/s; 2.5e8 bf16 ones in 300 tensors 1400, 8.0 GB at 5.7 TB/s (three launches of the norm and six of
// this, about 8 us each to drain and fill).  Division and square root are the correctly rounded ones; they hide behind the
// accesses.
template <typename T, bool STREAM>
__global__ __launch_bounds__(kThreads) void adamw(AdamTable tab, Clip clip, AdamArgs a, const float* steps) {
    constexpr bool kMaster = sizeof(T) == 2;
    constexpr int V = 4, kStep = kThreads * V;
    using P = Pack<T, V, STREAM>;
    using F = Pack<float, V, STREAM>;
    Factors f;
    if (clip.partials) {
        const double norm = norm_of(clip);
        if (blockIdx.x == 0 && threadIdx.x == 0 && clip.norm) *clip.norm = (float)norm;
        if (clip.skip_nonfinite && !isfinite((float)norm)) return;
        f.clip = coefficient(norm, clip.max_norm);
    }
    f.lr = a.lr_ptr ? *a.lr_ptr : a.lr;
    // lane i of each wave computes the factors of tensor i, ahead of the first chunk
    static_assert(AdamTable::kCap <= 64, "a lane per tensor");
    const int lane = threadIdx.x & 63;
    const float now = lane < tab.n ? steps[tab.id[lane]] + 1.f : 1.f;
    const float inv1 = 1.f / -expm1f((float)(now * a.ln1)), inv2 = 1.f / sqrtf(-expm1f((float)(now * a.ln2)));
    const int total = tab.end[tab.n - 1];
    Cursor<AdamTable::kCap> c(tab);
    T* p = nullptr;
    const T* g = nullptr;
    float *m = nullptr, *v = nullptr, *w = nullptr;
    for (int b = blockIdx.x; b < total; b += gridDim.x) {
        if (c.seek(tab, b)) {
            f.inv1 = of_lane(inv1, c.t);
            f.inv2 = of_lane(inv2, c.t);
            if (b == c.first && threadIdx.x == 0) *tab.step[c.t] = of_lane(now, c.t);
            p = (T*)tab.p[c.t];
            g = (const T*)tab.g[c.t];
            m = tab.m[c.t], v = tab.v[c.t], w = tab.w[c.t];
            c.align(tab, m);
        }
        c.range(tab, b);
        for (int64_t i = c.lo + threadIdx.x * V; i < c.hi; i += kStep) {
            if (i >= 0 && i + V <= c.hi) {
                typename P::type pi = P::load(p + i);
                const typename P::type gi = P::load(g + i);
                typename F::type mi = F::load(m + i), vi = F::load(v + i), wi = {};
                if (kMaster) wi = F::load(w + i);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float wj = kMaster ? weight_of<T>(pi[j], wi[j]) : (float)pi[j], mj = mi[j], vj = vi[j];
                    adamw_entry(wj, (float)gi[j], mj, vj, a, f);
                    if (kMaster) keep_rounded(wj);
                    wi[j] = wj, mi[j] = mj, vi[j] = vj, pi[j] = (T)wj;
                }
                P::store(p + i, pi);
                F::store(m + i, mi);
                F::store(v + i, vi);
                if (kMaster) F::store(w + i, wi);
            } else {
                for (int64_t j = i < 0 ? 0 : i; j < i + V && j < c.hi; ++j) {
                    float wj = kMaster ? weight_of<T>(p[j], w[j]) : (float)p[j], mj = m[j], vj = v[j];
                    adamw_entry(wj, (float)g[j], mj, vj, a, f);
                    if (kMaster) keep_rounded(wj);
                    m[j] = mj, v[j] = vj, p[j] = (T)wj;
                    if (kMaster) w[j] = wj;
                }
            }
        }
    }
}

// ---- host -------------------------------------------------------------------------------------------------------

bool known_dtype(int d) { return d == NERF_F32 || d == NERF_BF16 || d == NERF_F16; }
bool known_kind(int k) { return k == NERF_NORM_L1 || k == NERF_NORM_L2 || k == NERF_NORM_MAX; }
int elem_size(int d) { return d == NERF_F32 ? 4 : 2; }

int check_list(const void* const* ptr, const int64_t* numel, const int32_t* dtype, int n) {
    NERF_REQUIRE(n >= 0);
    NERF_REQUIRE(n == 0 || (ptr && numel && dtype));
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
        NERF_REQUIRE(numel[i] >= 0 && known_dtype(dtype[i]) && (ptr[i] || numel[i] == 0));
        if (numel[i] > ((int64_t)1 << 46) || (total += numel[i]) > ((int64_t)1 << 46)) return NERF_ERR_SIZE;
        NERF_REQUIRE((uintptr_t)ptr[i] % elem_size(dtype[i]) == 0);
    }
    return NERF_OK;
}

// Whether two of the tensors share memory (they are written by different workgroups).  Lists that ascend in memory,
// as the views of one buffer do, are seen in one pass; others are sorted.
int check_disjoint(void* const* ptr, const int64_t* numel, const int32_t* dtype, int n) {
    struct Span {
        uintptr_t lo, hi;
    };
    uintptr_t last = 0;
    bool ascending = true;
    for (int i = 0; i < n && ascending; ++i) {
        if (numel[i] == 0) continue;
        const uintptr_t lo = (uintptr_t)ptr[i];
        ascending = lo >= last;
        last = lo + numel[i] * elem_size(dtype[i]);
    }
    if (ascending) return NERF_OK;
    Span* s = (Span*)malloc(sizeof(Span) * n);
    if (!s) return NERF_ERR_SIZE;
    int k = 0;
    for (int i = 0; i < n; ++i)
        if (numel[i]) s[k++] = {(uintptr_t)ptr[i], (uintptr_t)ptr[i] + numel[i] * elem_size(dtype[i])};
    std::sort(s, s + k, [](const Span& a, const Span& b) { return a.lo < b.lo; });
    bool apart = true;
    for (int i = 1; i < k; ++i) apart = apart && s[i].lo >= s[i - 1].hi;
    free(s);
    return apart ? NERF_OK : NERF_ERR_ARG;
}

// ---- launches ---------------------------------------------------------------------------------------------------

// Elements per chunk of a list of `total`; beyond 2^30 chunks they get longer than `most`.
int chunk_for(int64_t total, const Cut& cut) {
    int64_t chunk = cut.least;
    while ((chunk < cut.most && total / chunk > cut.groups) || total / chunk > ((int64_t)1 << 30)) chunk *= 2;
    return (int)chunk;
}

int64_t list_elements(const int64_t* numel, int n) {
    int64_t total = 0;
    for (int i = 0; i < n; ++i) total += numel[i];
    return total;
}

int64_t list_bytes(const int64_t* numel, const int32_t* dtype, int n) {
    int64_t total = 0;
    for (int i = 0; i < n; ++i) total += numel[i] * elem_size(dtype[i]);
    return total;
}

// A launch leaves at most kNormGroups partials, and there are as many launches as full tables and one more per type.
int64_t max_partials(int n) { return (int64_t)kNormGroups * (3 + n / NormStepTable::kCap); }

struct Workspace {
    double* partials;
    float* steps;
};

int64_t workspace_bytes(int n) { return max_partials(n) * 8 + (int64_t)n * 4; }

int take_workspace(void* ws, int64_t bytes, int n, Workspace* out) {
    NERF_REQUIRE(ws && (uintptr_t)ws % 8 == 0 && bytes >= workspace_bytes(n));
    out->partials = (double*)ws;
    out->steps = (float*)(out->partials + max_partials(n));
    return NERF_OK;
}

// Tensors first .. last - 1 of a list of `total` elements, type by type: shift(i, element size) is shift_of its
// leading pointer; fill(k, i) puts it into place k of a table; go(type, workgroups) launches a full table, and the last of each
// type.  A tensor without elements has one empty chunk (its step counter still counts).
template <typename Table, typename Shift, typename Fill, typename Go>
void for_tables(Table& tab, Cut (*cut_of)(int), int64_t total, const int64_t* numel, const int32_t* dtype, int first, int last,
                Shift shift, Fill fill, Go go) {
    for (int d : {NERF_F32, NERF_BF16, NERF_F16}) {
        const Cut cut = cut_of(elem_size(d));
        tab.chunk = chunk_for(total, cut);
        tab.n = 0;
        int end = 0;
        for (int i = first; i < last; ++i) {
            if (dtype[i] != d) continue;
            const int64_t span = numel[i] + shift(i, elem_size(d));
            const int chunks = std::max(1, (int)((span + tab.chunk - 1) / tab.chunk));
            end += chunks;
            fill(tab.n, i);
            tab.end[tab.n] = end;
            tab.tail[tab.n] = (int)(span - (int64_t)(chunks - 1) * tab.chunk);
            if (++tab.n == Table::kCap) {
                go(d, std::min(end, cut.groups));
                tab.n = end = 0;
            }
        }
        if (tab.n) go(d, std::min(end, cut.groups));
    }
}

// go(element, streams) with values that carry the types of a kernel's instantiation.
template <typename Go>
void by_type(int d, bool streams, Go go) {
    const std::true_type yes;
    const std::false_type no;
    if (d == NERF_F32) streams ? go(float(), yes) : go(float(), no);
    else if (d == NERF_BF16) streams ? go(__bf16(), yes) : go(__bf16(), no);
    else streams ? go(_Float16(), yes) : go(_Float16(), no);
}

template <typename T, bool STREAM, typename Table>
void launch_norm(const Table& tab, int grid, int kind, double* partials, float* steps, hipStream_t st) {
    if (kind == NERF_NORM_L2) norm_partials<T, NERF_NORM_L2, STREAM><<<grid, kThreads, 0, st>>>(tab, partials, steps);
    else if (kind == NERF_NORM_L1) norm_partials<T, NERF_NORM_L1, STREAM><<<grid, kThreads, 0, st>>>(tab, partials, steps);
    else norm_partials<T, NERF_NORM_MAX, STREAM><<<grid, kThreads, 0, st>>>(tab, partials, steps);
}

// The norm's launches ahead of its reader's: a partial per workgroup -> how many.  more(k, i) fills what else the table
// holds.
template <bool CAN_STREAM, typename Table, typename More>
int run_norm(Table& tab, const void* const* ptr, const int64_t* numel, const int32_t* dtype, int n, int kind,
             const Workspace& ws, hipStream_t st, More more) {
    int partials = 0;
    const bool streams = CAN_STREAM && list_bytes(numel, dtype, n) > kNormStream;
    for_tables(tab, norm_cut, list_elements(numel, n), numel, dtype, 0, n,
               [&](int i, int size) { return shift_of(ptr[i], size); },
               [&](int k, int i) {
                   tab.ptr[k] = const_cast<void*>(ptr[i]);
                   more(k, i);
               },
               [&](int d, int grid) {
                   by_type(d, streams, [&](auto element, auto stream) {
                       launch_norm<decltype(element), CAN_STREAM && decltype(stream)::value>(
                           tab, grid, kind, ws.partials + partials, ws.steps, st);
                   });
                   partials += grid;
               });
    return partials;
}

}  // namespace

extern "C" int64_t nerf_grad_workspace_bytes(int n_tensors) { return n_tensors < 0 ? NERF_ERR_ARG : workspace_bytes(n_tensors); }

extern "C" int nerf_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtype, int n_tensors,
                              int norm_kind, void* workspace, int64_t n_workspace, float* norm, void* stream) {
    if (int e = check_list(grads, numel, dtype, n_tensors)) return e;
    NERF_REQUIRE(known_kind(norm_kind) && norm);
    Workspace ws;
    if (int e = take_workspace(workspace, n_workspace, n_tensors, &ws)) return e;
    hipStream_t st = nerf_stream(stream);
    ListTable tab;
    const int partials = run_norm<true>(tab, grads, numel, dtype, n_tensors, norm_kind, ws, st, [](int, int) {});
    norm_finish<<<1, kThreads, 0, st>>>(Clip{ws.partials, partials, norm_kind, 0, 0.0, norm});
    return nerf_launch_status();
}

extern "C" int nerf_clip_grad_norm(void* const* grads, const int64_t* numel, const int32_t* dtype, int n_tensors,
                                   int norm_kind, double max_norm, void* workspace, int64_t n_workspace, float* norm,
                                   void* stream) {
    if (int e = check_list(grads, numel, dtype, n_tensors)) return e;
    NERF_REQUIRE(known_kind(norm_kind) && max_norm >= 0.0 && norm);
    Workspace ws;
    if (int e = take_workspace(workspace, n_workspace, n_tensors, &ws)) return e;
    if (int e = check_disjoint(grads, numel, dtype, n_tensors)) return e;
    hipStream_t st = nerf_stream(stream);
    ListTable tab;
    const int partials = run_norm<false>(tab, grads, numel, dtype, n_tensors, norm_kind, ws, st, [](int, int) {});
    const Clip clip{ws.partials, partials, norm_kind, 0, max_norm, norm};
    if (n_tensors == 0) {
        norm_finish<<<1, kThreads, 0, st>>>(clip);
        return nerf_launch_status();
    }
    const bool streams = 2 * list_bytes(numel, dtype, n_tensors) > kUpdateStream;
    for_tables(tab, scale_cut, list_elements(numel, n_tensors), numel, dtype, 0, n_tensors,
               [&](int i, int size) { return shift_of(grads[i], size); }, [&](int k, int i) { tab.ptr[k] = grads[i]; },
               [&](int d, int grid) {
                   by_type(d, streams, [&](auto element, auto s) {
                       scale_by_norm<decltype(element), decltype(s)::value><<<grid, kThreads, 0, st>>>(tab, clip);
                   });
               });
    return nerf_launch_status();
}

extern "C" int nerf_adamw_step(const nerf_adamw_tensors* t, const nerf_adamw_group* groups, int n_groups, int norm_kind,
                               double max_norm, int skip_nonfinite, void* workspace, int64_t n_workspace, float* norm,
                               void* stream) {
    NERF_REQUIRE(t && n_groups >= 0 && (groups || n_groups == 0));
    const int n = t->n_tensors;
    if (int e = check_list(t->param, t->numel, t->dtype, n)) return e;
    if (int e = check_list(t->grad, t->numel, t->dtype, n)) return e;
    NERF_REQUIRE(n == 0 || (t->exp_avg && t->exp_avg_sq && t->step));
    int covered = 0;
    for (int i = 0; i < n; ++i) {
        const bool half = t->dtype[i] != NERF_F32;
        NERF_REQUIRE(t->step[i] && (uintptr_t)t->step[i] % 4 == 0);
        NERF_REQUIRE(!half || t->master);
        if (t->numel[i] == 0) continue;
        NERF_REQUIRE(t->exp_avg[i] && t->exp_avg_sq[i] && (!half || t->master[i]));
        NERF_REQUIRE(((uintptr_t)t->exp_avg[i] | (uintptr_t)t->exp_avg_sq[i]) % 4 == 0);
        NERF_REQUIRE(!half || (uintptr_t)t->master[i] % 4 == 0);
    }
    for (int k = 0; k < n_groups; ++k) {
        const nerf_adamw_group& g = groups[k];
        NERF_REQUIRE(g.count >= 0 && g.count <= n - covered);
        NERF_REQUIRE(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0 && g.eps >= 0.0);
        covered += g.count;
    }
    NERF_REQUIRE(covered == n);
    const bool clips = norm_kind != NERF_NORM_NONE;
    NERF_REQUIRE(!clips || (known_kind(norm_kind) && max_norm >= 0.0));
    NERF_REQUIRE(clips || !skip_nonfinite);
    if (n == 0) {
        if (!clips || !norm) return NERF_OK;
        norm_finish<<<1, kThreads, 0, nerf_stream(stream)>>>(Clip{nullptr, 0, norm_kind, 0, 0.0, norm});
        return nerf_launch_status();
    }
    Workspace ws;
    if (int e = take_workspace(workspace, n_workspace, n, &ws)) return e;
    if (int e = check_disjoint(t->param, t->numel, t->dtype, n)) return e;
    hipStream_t st = nerf_stream(stream);
    Clip clip{nullptr, 0, norm_kind, skip_nonfinite, max_norm, norm};
    // The step counters are read ahead of the update, in a launch of their own (the norm's, if there is one): in the
    // update the first workgroup of a tensor writes a counter that the others of that tensor need the old value of.
    if (clips) {
        clip.partials = ws.partials;
        NormStepTable norms;
        clip.n_partials = run_norm<false>(norms, t->grad, t->numel, t->dtype, n, norm_kind, ws, st, [&](int k, int i) {
            norms.step[k] = t->step[i];
            norms.id[k] = i;
        });
    } else {
        StepTable s;
        for (s.first_tensor = 0; s.first_tensor < n; s.first_tensor += s.n) {
            for (s.n = 0; s.n < kStepCap && s.first_tensor + s.n < n; ++s.n) s.step[s.n] = t->step[s.first_tensor + s.n];
            read_steps<<<1, kThreads, 0, st>>>(s, ws.steps);
        }
    }
    const int64_t elements = list_elements(t->numel, n);
    const bool streams = 28 * elements > kUpdateStream;
    AdamTable tab;
    int first = 0;
    for (int k = 0; k < n_groups; ++k) {
        const nerf_adamw_group& g = groups[k];
        const AdamArgs a{g.lr_device,          (float)g.lr,           (float)g.beta1, (float)g.beta2, (float)g.eps,
                         (float)g.weight_decay, (float)(1.0 - g.beta1), (float)(1.0 - g.beta2), log(g.beta1), log(g.beta2)};
        for_tables(tab, adam_cut, elements, t->numel, t->dtype, first, first + g.count,
                   [&](int i, int) { return shift_of(t->exp_avg[i], 4); },
                   [&](int j, int i) {
                       tab.p[j] = t->param[i];
                       tab.g[j] = t->grad[i];
                       tab.m[j] = t->exp_avg[i];
                       tab.v[j] = t->exp_avg_sq[i];
                       tab.w[j] = t->master ? t->master[i] : nullptr;
                       tab.step[j] = t->step[i];
                       tab.id[j] = i;
                   },
                   [&](int d, int grid) {
                       by_type(d, streams, [&](auto element, auto s) {
                           adamw<decltype(element), decltype(s)::value><<<grid, kThreads, 0, st>>>(tab, clip, a, ws.steps);
                       });
                   });
        first += g.count;
    }
    return nerf_launch_status();
}
