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
// several launches.  Each tensor is cut into chunks, one workgroup per chunk.  The norm is one launch that leaves a
// partial sum per chunk in the caller's workspace; every workgroup of the launch that needs the norm adds those up for
// itself, in one fixed order, so that there are no atomics, no waiting between workgroups, no launch in between, and
// the same bits on every call.
#include <stdlib.h>

#include <algorithm>
#include <cmath>

#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kNormCap = 128;       // tensors per launch: the tables stay below 4 KB of kernel arguments
constexpr int kScaleCap = 128;
constexpr int kAdamCap = 64;
constexpr int kStepCap = 256;
constexpr int kMaxPartials = 2048;  // chunks of one call: at most this many, and one more per tensor
constexpr int kMinChunk = 1024;

struct NormTable {
    const void* ptr[kNormCap];
    const float* step[kNormCap];    // null, or the tensor's step counter: copied to the workspace
    int64_t numel[kNormCap];
    int end[kNormCap];              // chunks of the tensors up to and including this one
    int n, first_tensor, first_partial;
    int64_t chunk;
};

struct ScaleTable {
    void* ptr[kScaleCap];
    int64_t numel[kScaleCap];
    int end[kScaleCap];
    int n;
    int64_t chunk;
};

struct AdamTable {
    void* p[kAdamCap];
    const void* g[kAdamCap];
    float* m[kAdamCap];
    float* v[kAdamCap];
    float* w[kAdamCap];             // 32-bit master weights (16-bit parameters)
    float* step[kAdamCap];
    int64_t numel[kAdamCap];
    int end[kAdamCap];
    int n, first_tensor;
    int64_t chunk;
};

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
    float lr, beta2, eps, decay, rest1, rest2;      // rest = 1 - beta, rounded from 64 bits
    float beta1;
    double ln1, ln2;                // ln(beta)
};

// The table entry that a chunk belongs to.  The lanes of a wave compare 64 entries at a time: two loads deep, where a
// bisection through the kernel's arguments would be six or seven.
template <int CAP>
__device__ __forceinline__ int find_tensor(const int (&end)[CAP], int n, int chunk) {
    int idx = 0;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int base = 0; base < CAP; base += 64) {
        const int i = base + lane;
        idx += __popcll(__ballot(i < n && end[i < n ? i : 0] <= chunk));
    }
    return __builtin_amdgcn_readfirstlane(idx);
}

// ---- sums in a fixed order --------------------------------------------------------------------------------------
// Sums are held in 64 bits: the square of a 32-bit value is exact there, and neither overflows nor underflows, so the
// norm needs no scaling pass.  Maxima compare the bits of the absolute value, under which a NaN is the largest.

template <int KIND>
__device__ __forceinline__ double join(double a, double b) {
    if (KIND != NERF_NORM_MAX) return a + b;
    return __double_as_longlong(a) > __double_as_longlong(b) ? a : b;
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
    double x = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) x = join<KIND>(x, partials[i]);
    x = group_join<KIND>(x);
    return KIND == NERF_NORM_L2 ? sqrt(x) : x;
}

__device__ __forceinline__ double norm_of(const Clip& c) {
    if (c.kind == NERF_NORM_L2) return norm_of<NERF_NORM_L2>(c.partials, c.n_partials);
    if (c.kind == NERF_NORM_L1) return norm_of<NERF_NORM_L1>(c.partials, c.n_partials);
    return norm_of<NERF_NORM_MAX>(c.partials, c.n_partials);
}

__device__ __forceinline__ float coefficient(double norm, double max_norm) {
    const double d = norm + 1e-6;
    return d <= max_norm ? 1.f : (float)(max_norm / d);       // (a NaN norm gives NaN)
}

template <typename T, int KIND>
__global__ __launch_bounds__(kThreads) void norm_partials(NormTable tab, double* partials, float* steps) {
    const int b = blockIdx.x;
    const int t = find_tensor(tab.end, tab.n, b);
    const int first = t ? tab.end[t - 1] : 0;
    const T* g = (const T*)tab.ptr[t];
    const int64_t lo = (int64_t)(b - first) * tab.chunk;
    const int64_t hi = lo + tab.chunk < tab.numel[t] ? lo + tab.chunk : tab.numel[t];
    double acc = 0.0;
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) {
        const float x = (float)g[i];
        if (KIND == NERF_NORM_L2) acc = fma((double)x, (double)x, acc);
        else acc = join<KIND>(acc, (double)fabsf(x));
    }
    acc = group_join<KIND>(acc);
    if (threadIdx.x == 0) {
        partials[tab.first_partial + b] = acc;
        if (b == first && tab.step[t]) steps[tab.first_tensor + t] = *tab.step[t];
    }
}

__global__ __launch_bounds__(kThreads) void norm_finish(Clip clip) {
    const double n = norm_of(clip);
    if (threadIdx.x == 0) *clip.norm = (float)n;
}

__global__ __launch_bounds__(kThreads) void read_steps(StepTable tab, float* steps) {
    const int i = threadIdx.x;
    if (i < tab.n) steps[tab.first_tensor + i] = *tab.step[i];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void scale_by_norm(ScaleTable tab, Clip clip) {
    const int b = blockIdx.x;
    const int t = find_tensor(tab.end, tab.n, b);
    const int first = t ? tab.end[t - 1] : 0;
    const double norm = norm_of(clip);
    if (b == 0 && threadIdx.x == 0 && clip.norm) *clip.norm = (float)norm;
    const float c = coefficient(norm, clip.max_norm);
    T* g = (T*)tab.ptr[t];
    const int64_t lo = (int64_t)(b - first) * tab.chunk;
    const int64_t hi = lo + tab.chunk < tab.numel[t] ? lo + tab.chunk : tab.numel[t];
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) g[i] = (T)((float)g[i] * c);
}

// A 16-bit parameter is the rounding of its 32-bit master.  Left to itself the compiler forms the last multiply-add
// and the conversion to fp16 as one instruction, which rounds the exact sum once and so may end on the other neighbour
// than the rounding of the rounded sum: the value has to exist in 32 bits first.
__device__ __forceinline__ void keep_rounded(float& x) { asm("" : "+v"(x)); }

template <typename T>
__global__ __launch_bounds__(kThreads) void adamw(AdamTable tab, Clip clip, AdamArgs a, const float* steps) {
    constexpr bool kMaster = sizeof(T) == 2;
    const int b = blockIdx.x;
    const int t = find_tensor(tab.end, tab.n, b);
    const int first = t ? tab.end[t - 1] : 0;
    float c = 1.f;
    if (clip.partials) {
        const double norm = norm_of(clip);
        if (b == 0 && tab.first_tensor == 0 && threadIdx.x == 0 && clip.norm) *clip.norm = (float)norm;
        if (clip.skip_nonfinite && !isfinite((float)norm)) return;
        c = coefficient(norm, clip.max_norm);
    }
    const float now = steps[tab.first_tensor + t] + 1.f;
    if (b == first && threadIdx.x == 0) *tab.step[t] = now;
    const float lr = a.lr_ptr ? *a.lr_ptr : a.lr;
    const float inv1 = 1.f / -expm1f((float)(now * a.ln1));             // 1 / (1 - beta^t)
    const float inv2 = 1.f / sqrtf(-expm1f((float)(now * a.ln2)));
    T* p = (T*)tab.p[t];
    const T* g = (const T*)tab.g[t];
    float *m = tab.m[t], *v = tab.v[t], *w = tab.w[t];
    const int64_t lo = (int64_t)(b - first) * tab.chunk;
    const int64_t hi = lo + tab.chunk < tab.numel[t] ? lo + tab.chunk : tab.numel[t];
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) {
        const float gi = (float)g[i] * c;
        const float mi = a.beta1 * m[i] + a.rest1 * gi;
        const float vi = a.beta2 * v[i] + a.rest2 * (gi * gi);
        const T pi = p[i];
        float wi = (float)pi;
        if (kMaster) {
            // the master stands for the parameter as long as it rounds to it: a parameter that was written from
            // outside (a loaded checkpoint) is taken as it is
            const float wm = w[i];
            if ((T)wm == pi) wi = wm;
        }
        wi -= lr * (mi * inv1 / (sqrtf(vi) * inv2 + a.eps) + a.decay * wi);
        if (kMaster) keep_rounded(wi);
        m[i] = mi;
        v[i] = vi;
        p[i] = (T)wi;
        if (kMaster) w[i] = wi;
    }
}

// ---- host -------------------------------------------------------------------------------------------------------

bool known_dtype(int d) { return d == NERF_F32 || d == NERF_BF16 || d == NERF_F16; }
bool known_kind(int k) { return k == NERF_NORM_L1 || k == NERF_NORM_L2 || k == NERF_NORM_MAX; }
int64_t elem_size(int d) { return d == NERF_F32 ? 4 : 2; }

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

// Elements per chunk: as few as kMinChunk while the list is short (latency: every compute unit gets some), more once
// there would be more than kMaxPartials chunks.
int64_t chunk_for(const int64_t* numel, int n) {
    int64_t total = 0;
    for (int i = 0; i < n; ++i) total += numel[i];
    int64_t chunk = kMinChunk;
    while ((total + chunk - 1) / chunk > kMaxPartials) chunk *= 2;
    return chunk;
}

// a tensor without elements has one empty chunk (its step counter still counts)
int chunks_of(int64_t numel, int64_t chunk) { return numel ? (int)((numel + chunk - 1) / chunk) : 1; }

struct Workspace {
    double* partials;
    float* steps;
};

int64_t workspace_bytes(int n) { return (int64_t)(kMaxPartials + n) * 8 + (int64_t)n * 4; }

int take_workspace(void* ws, int64_t bytes, int n, Workspace* out) {
    NERF_REQUIRE(ws && (uintptr_t)ws % 8 == 0 && bytes >= workspace_bytes(n));
    out->partials = (double*)ws;
    out->steps = (float*)(out->partials + kMaxPartials + n);
    return NERF_OK;
}

template <typename T>
void launch_norm(const NormTable& tab, int kind, const Workspace& ws, hipStream_t st) {
    const dim3 grid(tab.end[tab.n - 1]), block(kThreads);
    if (kind == NERF_NORM_L2) norm_partials<T, NERF_NORM_L2><<<grid, block, 0, st>>>(tab, ws.partials, ws.steps);
    else if (kind == NERF_NORM_L1) norm_partials<T, NERF_NORM_L1><<<grid, block, 0, st>>>(tab, ws.partials, ws.steps);
    else norm_partials<T, NERF_NORM_MAX><<<grid, block, 0, st>>>(tab, ws.partials, ws.steps);
}

// The norm's first launch(es): a partial per chunk.  Tables hold consecutive tensors of one type.
int run_norm(const void* const* ptr, float* const* step, const int64_t* numel, const int32_t* dtype, int n, int kind,
             const Workspace& ws, int* n_partials, hipStream_t st) {
    const int64_t chunk = chunk_for(numel, n);
    NormTable tab;
    tab.chunk = chunk;
    int partials = 0;
    for (int i = 0; i < n;) {
        const int d = dtype[i];
        tab.n = 0;
        tab.first_tensor = i;
        tab.first_partial = partials;
        int end = 0;
        for (; i < n && tab.n < kNormCap && dtype[i] == d; ++i, ++tab.n) {
            end += chunks_of(numel[i], chunk);
            tab.ptr[tab.n] = ptr[i];
            tab.step[tab.n] = step ? step[i] : nullptr;
            tab.numel[tab.n] = numel[i];
            tab.end[tab.n] = end;
        }
        partials += end;
        if (d == NERF_F32) launch_norm<float>(tab, kind, ws, st);
        else if (d == NERF_BF16) launch_norm<__bf16>(tab, kind, ws, st);
        else launch_norm<_Float16>(tab, kind, ws, st);
    }
    *n_partials = partials;
    return nerf_launch_status();
}

}  // namespace

extern "C" int64_t nerf_grad_workspace_bytes(int n_tensors) { return n_tensors < 0 ? NERF_ERR_ARG : workspace_bytes(n_tensors); }

extern "C" int nerf_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtype, int n_tensors,
                              int norm_kind, void* workspace, int64_t workspace_bytes_, float* norm, void* stream) {
    if (int e = check_list(grads, numel, dtype, n_tensors)) return e;
    NERF_REQUIRE(known_kind(norm_kind) && norm);
    Workspace ws;
    if (int e = take_workspace(workspace, workspace_bytes_, n_tensors, &ws)) return e;
    int partials = 0;
    if (int e = run_norm(grads, nullptr, numel, dtype, n_tensors, norm_kind, ws, &partials, nerf_stream(stream))) return e;
    norm_finish<<<1, kThreads, 0, nerf_stream(stream)>>>(Clip{ws.partials, partials, norm_kind, 0, 0.0, norm});
    return nerf_launch_status();
}

extern "C" int nerf_clip_grad_norm(void* const* grads, const int64_t* numel, const int32_t* dtype, int n_tensors,
                                   int norm_kind, double max_norm, void* workspace, int64_t workspace_bytes_, float* norm,
                                   void* stream) {
    if (int e = check_list(grads, numel, dtype, n_tensors)) return e;
    NERF_REQUIRE(known_kind(norm_kind) && max_norm >= 0.0 && norm);
    Workspace ws;
    if (int e = take_workspace(workspace, workspace_bytes_, n_tensors, &ws)) return e;
    if (int e = check_disjoint(grads, numel, dtype, n_tensors)) return e;
    hipStream_t st = nerf_stream(stream);
    int partials = 0;
    if (int e = run_norm(grads, nullptr, numel, dtype, n_tensors, norm_kind, ws, &partials, st)) return e;
    const Clip clip{ws.partials, partials, norm_kind, 0, max_norm, norm};
    if (n_tensors == 0) {
        norm_finish<<<1, kThreads, 0, st>>>(clip);
        return nerf_launch_status();
    }
    ScaleTable tab;
    tab.chunk = chunk_for(numel, n_tensors);
    for (int i = 0; i < n_tensors;) {
        const int d = dtype[i];
        int end = 0;
        tab.n = 0;
        for (; i < n_tensors && tab.n < kScaleCap && dtype[i] == d; ++i, ++tab.n) {
            end += chunks_of(numel[i], tab.chunk);
            tab.ptr[tab.n] = grads[i];
            tab.numel[tab.n] = numel[i];
            tab.end[tab.n] = end;
        }
        if (d == NERF_F32) scale_by_norm<float><<<end, kThreads, 0, st>>>(tab, clip);
        else if (d == NERF_BF16) scale_by_norm<__bf16><<<end, kThreads, 0, st>>>(tab, clip);
        else scale_by_norm<_Float16><<<end, kThreads, 0, st>>>(tab, clip);
    }
    return nerf_launch_status();
}

extern "C" int nerf_adamw_step(const nerf_adamw_tensors* t, const nerf_adamw_group* groups, int n_groups, int norm_kind,
                               double max_norm, int skip_nonfinite, void* workspace, int64_t workspace_bytes_, float* norm,
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
    if (n == 0) return NERF_OK;
    Workspace ws;
    if (int e = take_workspace(workspace, workspace_bytes_, n, &ws)) return e;
    if (int e = check_disjoint(t->param, t->numel, t->dtype, n)) return e;
    hipStream_t st = nerf_stream(stream);
    Clip clip{nullptr, 0, norm_kind, skip_nonfinite, max_norm, norm};
    // The step counters are read ahead of the update, in a launch of their own (the norm's, if there is one): in the
    // update the first workgroup of a tensor writes a counter that the others of that tensor need the old value of.
    if (clips) {
        clip.partials = ws.partials;
        if (int e = run_norm(t->grad, t->step, t->numel, t->dtype, n, norm_kind, ws, &clip.n_partials, st)) return e;
    } else {
        StepTable s;
        for (s.first_tensor = 0; s.first_tensor < n; s.first_tensor += s.n) {
            for (s.n = 0; s.n < kStepCap && s.first_tensor + s.n < n; ++s.n) s.step[s.n] = t->step[s.first_tensor + s.n];
            read_steps<<<1, kThreads, 0, st>>>(s, ws.steps);
        }
    }
    AdamTable tab;
    tab.chunk = chunk_for(t->numel, n);
    int i = 0, group_end = 0;
    for (int k = 0; k < n_groups; ++k) {
        const nerf_adamw_group& g = groups[k];
        group_end += g.count;
        const AdamArgs a{g.lr_device, (float)g.lr, (float)g.beta2, (float)g.eps, (float)g.weight_decay, (float)(1.0 - g.beta1),
                         (float)(1.0 - g.beta2), (float)g.beta1, log(g.beta1), log(g.beta2)};
        while (i < group_end) {
            const int d = t->dtype[i];
            int end = 0;
            tab.n = 0;
            tab.first_tensor = i;
            for (; i < group_end && tab.n < kAdamCap && t->dtype[i] == d; ++i, ++tab.n) {
                end += chunks_of(t->numel[i], tab.chunk);
                tab.p[tab.n] = t->param[i];
                tab.g[tab.n] = t->grad[i];
                tab.m[tab.n] = t->exp_avg[i];
                tab.v[tab.n] = t->exp_avg_sq[i];
                tab.w[tab.n] = t->master ? t->master[i] : nullptr;
                tab.step[tab.n] = t->step[i];
                tab.numel[tab.n] = t->numel[i];
                tab.end[tab.n] = end;
            }
            if (d == NERF_F32) adamw<float><<<end, kThreads, 0, st>>>(tab, clip, a, ws.steps);
            else if (d == NERF_BF16) adamw<__bf16><<<end, kThreads, 0, st>>>(tab, clip, a, ws.steps);
            else adamw<_Float16><<<end, kThreads, 0, st>>>(tab, clip, a, ws.steps);
        }
    }
    return nerf_launch_status();
}
