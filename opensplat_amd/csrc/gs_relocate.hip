// gs_relocate.hip — target Gaussians become copies of drawn source Gaussians.  C ABI: include/gsplat_densify.h
// (gs_relocate), which also holds the definition.
//
// A source that is copied c times becomes m = c + 1 equal Gaussians that together look like the one that was there:
//   opacity   1 - (1 - o')^m = o:   with y = softplus(logit) / m, o' = 1 - exp(-y) and logit' = log(expm1(y))
//   extent    the integral of 1 - (1 - o' exp(-t^2 / 2s'^2))^m over the line equals o times the Gaussian's own; expanding the
//             power, s' = s o / D,  D = sum_{j=1..m} (-1)^(j-1) C(m, j) o'^j / sqrt(j)
// C(m, j) o'^j <= Y^j / j! with Y = softplus(logit) <= 16 (the logit is clamped there), so the alternating sum converges
// within 96 terms whatever m is; in 64 bits its cancellation (terms up to e^Y, some forty roundings in each) costs an
// absolute 1e-7 at the clamp and 1e-10 for logits below 9, where a float's own rounding is 6e-8.
//
//   k_relocate_clear   the words of the rows that are named: owner, copies
//   k_relocate_claim   a target belongs to the first pair that names it; every target of a pair in range is marked
//   k_relocate_count   pairs that hold (own target, source that is no target) are counted per source; the pair that is
//                      counted first also rewrites the source — which one that is changes no result
//   k_relocate_rows    64 pairs per workgroup: one lane each for opacity and extent, then their rows, a wave per pair
// A source's opacity and scales are rewritten by one workgroup while others may hold pairs of the same source: those
// columns are read by k_relocate_count, which writes no row, and kept per pair; k_relocate_rows reads only columns that
// stay as they are.
#include <math.h>

#include "gs_device.h"
#include "../../include/gsplat_densify.h"

namespace gs {

constexpr int kRelThreads = 256;
constexpr int kRelTerms = 96;
constexpr int32_t kNoOwner = 0x7fffffff;

struct RelocatePair {
    float logit, s0, s1, s2;                   // the source's, before
    int32_t rank;                              // order among the source's pairs, -1: the pair does not hold
};

static __device__ __forceinline__ bool in_range(int32_t i, int N) { return i >= 0 && i < N; }

__global__ void __launch_bounds__(kRelThreads)
k_relocate_clear(int N, int pairs, const int32_t *__restrict__ targets, const int32_t *__restrict__ sources,
                 int32_t *__restrict__ owner, int32_t *__restrict__ copies) {
    const int i = blockIdx.x * kRelThreads + threadIdx.x;
    if (i >= pairs) return;
    const int32_t t = targets[i], s = sources[i];
    if (!in_range(t, N) || !in_range(s, N)) return;
    owner[t] = kNoOwner;
    owner[s] = kNoOwner;
    copies[s] = 0;
}

__global__ void __launch_bounds__(kRelThreads)
k_relocate_claim(int N, int pairs, const int32_t *__restrict__ targets, const int32_t *__restrict__ sources,
                 int32_t *__restrict__ owner) {
    const int i = blockIdx.x * kRelThreads + threadIdx.x;
    if (i >= pairs) return;
    const int32_t t = targets[i], s = sources[i];
    if (in_range(t, N) && in_range(s, N)) atomicMin(&owner[t], i);
}

__global__ void __launch_bounds__(kRelThreads)
k_relocate_count(int N, int pairs, const int32_t *__restrict__ targets, const int32_t *__restrict__ sources,
                 const int32_t *__restrict__ owner, int32_t *__restrict__ copies, const float *__restrict__ logits,
                 const float *__restrict__ log_scales, RelocatePair *__restrict__ out) {
    const int i = blockIdx.x * kRelThreads + threadIdx.x;
    if (i >= pairs) return;
    const int32_t t = targets[i], s = sources[i];
    RelocatePair p = {0.0f, 0.0f, 0.0f, 0.0f, -1};
    if (in_range(t, N) && in_range(s, N) && owner[t] == i && owner[s] == kNoOwner) {
        p.logit = logits[s];
        p.s0 = log_scales[3 * (size_t)s];
        p.s1 = log_scales[3 * (size_t)s + 1];
        p.s2 = log_scales[3 * (size_t)s + 2];
        p.rank = atomicAdd(&copies[s], 1);
    }
    out[i] = p;
}

struct RelocateSets {
    float *p[6], *m[6], *v[6];
    int rest_len;
};

// log(o / D) and the new logit of a source with `m` equal shares
static __device__ __forceinline__ void share(float logit, int m, double min_logit, float &new_logit, float &shrink) {
    const double x = fmin((double)logit, 16.0);
    const double big = (x > 0.0 ? x + log1p(exp(-x)) : log1p(exp(x)));   // softplus = -log(1 - o)
    const double y = big / (double)m, p = -expm1(-y);
    double term = 1.0, sum = 0.0;
    for (int j = 1; j <= kRelTerms && j <= m; j++) {
        term *= (double)(m - j + 1) / (double)j * p;
        const double t = term / sqrt((double)j);
        sum += (j & 1) ? t : -t;
        if (term < 1e-18 * sum) break;
    }
    const double log_o = x < 0.0 ? x - log1p(exp(x)) : -log1p(exp(-x));
    new_logit = (float)fmax(log(expm1(y)), min_logit);
    shrink = (float)(log_o - log(sum));
}

__global__ void __launch_bounds__(kRelThreads)
k_relocate_rows(int pairs, const int32_t *__restrict__ targets, const int32_t *__restrict__ sources,
                const int32_t *__restrict__ copies, const RelocatePair *__restrict__ in, double min_logit,
                RelocateSets a) {
    __shared__ float4 fresh[64];               // new logit, new log-scales
    __shared__ int32_t rank[64];
    const int tid = threadIdx.x, first = blockIdx.x * 64;
    if (tid < 64) {
        const int i = first + tid;
        rank[tid] = -1;
        if (i < pairs) {
            const RelocatePair p = in[i];
            rank[tid] = p.rank;
            if (p.rank >= 0) {
                float l, d;
                share(p.logit, copies[sources[i]] + 1, min_logit, l, d);
                fresh[tid] = make_float4(l, p.s0 + d, p.s1 + d, p.s2 + d);
            }
        }
    }
    __syncthreads();
    const int lane = tid & 63;
    for (int k = tid >> 6; k < 64; k += kRelThreads / 64) {
        const int rk = rank[k];
        if (rk < 0) continue;
        const size_t t = (size_t)targets[first + k], s = (size_t)sources[first + k];
        const float4 f = fresh[k];
        const int lens[6] = {3, 3, 4, 1, 3, a.rest_len};
        for (int q = 0; q < 6; q++) {
            const int len = lens[q];
            for (int c = lane; c < len; c += 64) {
                float v;
                if (q == 1) v = c == 0 ? f.y : (c == 1 ? f.z : f.w);
                else if (q == 3) v = f.x;
                else v = a.p[q][s * len + c];
                a.p[q][t * len + c] = v;
                if (rk == 0 && (q == 1 || q == 3)) a.p[q][s * len + c] = v;
                if (a.m[q]) {
                    a.m[q][t * len + c] = 0.0f;
                    if (rk == 0) a.m[q][s * len + c] = 0.0f;
                }
                if (a.v[q]) {
                    a.v[q][t * len + c] = 0.0f;
                    if (rk == 0) a.v[q][s * len + c] = 0.0f;
                }
            }
        }
    }
}

struct RelocateLayout {
    size_t owner_off, copies_off, pairs_off, total;
    RelocateLayout(int N, int pairs) {
        size_t o = 0;
        auto take = [&](size_t bytes) { size_t r = o; o += (bytes + 255) & ~(size_t)255; return r; };
        owner_off = take((size_t)N * 4);
        copies_off = take((size_t)N * 4);
        pairs_off = take((size_t)pairs * sizeof(RelocatePair));
        total = o;
    }
};

}  // namespace gs

extern "C" size_t gs_relocate_workspace_bytes(int N, int pairs) {
    if (N <= 0 || pairs < 0) return 0;
    return gs::RelocateLayout(N, pairs).total;
}

extern "C" int gs_relocate(int N, int K, int pairs, const int32_t *targets, const int32_t *sources, float min_opacity,
                           const GsGaussianSet *params, const GsGaussianSet *exp_avg, const GsGaussianSet *exp_avg_sq,
                           void *workspace, size_t workspace_bytes, gs_stream_t stream) {
    using namespace gs;
    if (N <= 0 || K < 1 || pairs < 0 || !params || !(min_opacity > 0.0f && min_opacity < 1.0f))
        return GS_ERR_INVALID_ARGUMENT;
    if (pairs == 0) return GS_OK;
    if (!targets || !sources || !workspace || ((uintptr_t)workspace & 15)) return GS_ERR_INVALID_ARGUMENT;
    const GsGaussianSet none = {nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
    const GsGaussianSet &p = *params, &m = exp_avg ? *exp_avg : none, &v = exp_avg_sq ? *exp_avg_sq : none;
    if (!p.means || !p.log_scales || !p.quats || !p.opacity_logits || !p.features_dc || (K > 1 && !p.features_rest))
        return GS_ERR_INVALID_ARGUMENT;
    const RelocateLayout L(N, pairs);
    if (workspace_bytes < L.total) return GS_ERR_WORKSPACE;
    char *ws = (char *)workspace;
    int32_t *owner = (int32_t *)(ws + L.owner_off), *copies = (int32_t *)(ws + L.copies_off);
    RelocatePair *held = (RelocatePair *)(ws + L.pairs_off);
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((pairs + kRelThreads - 1) / kRelThreads), block(kRelThreads);
    GS_LAUNCH(k_relocate_clear, grid, block, 0, s, N, pairs, targets, sources, owner, copies);
    GS_LAUNCH_CHECK();
    GS_LAUNCH(k_relocate_claim, grid, block, 0, s, N, pairs, targets, sources, owner);
    GS_LAUNCH_CHECK();
    GS_LAUNCH(k_relocate_count, grid, block, 0, s, N, pairs, targets, sources, owner, copies, p.opacity_logits,
              p.log_scales, held);
    GS_LAUNCH_CHECK();
    RelocateSets a = {{p.means, p.log_scales, p.quats, p.opacity_logits, p.features_dc, p.features_rest},
                      {m.means, m.log_scales, m.quats, m.opacity_logits, m.features_dc, m.features_rest},
                      {v.means, v.log_scales, v.quats, v.opacity_logits, v.features_dc, v.features_rest},
                      (K - 1) * 3};
    const double o = (double)min_opacity;
    GS_LAUNCH(k_relocate_rows, dim3((pairs + 63) / 64), block, 0, s, pairs, targets, sources, copies, held,
              log(o / (1.0 - o)), a);
    GS_LAUNCH_CHECK();
    return GS_OK;
}
