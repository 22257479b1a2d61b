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
//   k_relocate_few     these three, where pairs are few
//   k_relocate_rows    16 pairs per workgroup: one lane each for opacity and extent, then their rows, a wave for four pairs
//                      with a lane per column of the six tensors, so that a row is one load and its copy one store
// A source's opacity and scales are rewritten by one workgroup while others may hold pairs of the same source: those
// columns are read by k_relocate_count, which writes no row, and kept per pair; k_relocate_rows reads only columns that
// stay as they are.
//
// Bound by scattered lines: a row of 59 floats lies in six places (some nine 64-byte lines), written for the copy in
// parameters and moments, and in the moments for the source: some 56 lines a pair.  Measured: 300 pairs 5.3 + 6.6 us, 50 000
// of a million Gaussians 19 + 39 us from the caches; a call on rows that are not in them 100 us, where 56 lines a pair are 37 at
// a copy's rate: a row's loads stand behind its pair's opacity and extent, the moments' zeros behind the loads.
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

// The three of them for few pairs, as one workgroup's phases, a pair a thread (launches of a microsecond of work cost the host
// two each).  Its one compute unit's loads and atomics grow with the pairs: calls of 300 pairs 15.6 us against 21.5 in three
// launches, 640 17.8 and 21.6, 1000 22.9 and 21.8 (2000, two pairs a thread, 38 and 22).
// The words pass through the device's atomics: a load of this unit's own cache could be older.
constexpr int kFewPairs = 768;
__global__ void __launch_bounds__(kFewPairs)
k_relocate_few(int N, int pairs, const int32_t *__restrict__ targets, const int32_t *__restrict__ sources, int32_t *owner,
               int32_t *copies, const float *__restrict__ logits, const float *__restrict__ log_scales,
               RelocatePair *__restrict__ out) {
    const int i = threadIdx.x;
    int32_t t = -1, s = -1;
    if (i < pairs) {
        t = targets[i];
        s = sources[i];
    }
    const bool valid = in_range(t, N) && in_range(s, N);
    if (valid) {
        __hip_atomic_store(&owner[t], kNoOwner, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&owner[s], kNoOwner, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&copies[s], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (valid) atomicMin(&owner[t], i);
    __syncthreads();
    RelocatePair p = {0.0f, 0.0f, 0.0f, 0.0f, -1};
    if (valid && __hip_atomic_load(&owner[t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == i &&
        __hip_atomic_load(&owner[s], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == kNoOwner) {
        p.logit = logits[s];
        p.s0 = log_scales[3 * (size_t)s];
        p.s1 = log_scales[3 * (size_t)s + 1];
        p.s2 = log_scales[3 * (size_t)s + 2];
        p.rank = atomicAdd(&copies[s], 1);
    }
    if (i < pairs) out[i] = p;
}

struct RelocateSets {
    float *p[6], *m[6], *v[6];
    int columns;                               // floats per Gaussian over the six tensors
};

constexpr int kRowPairs = 16;

// log(o / D) and the new logit of a source with `m` equal shares; `inverse` [j] = {1 / j, 1 / sqrt(j)}.
// Below e^-40 what the sums differ by from their first terms is less than a rounding: o' = o / m, D = o, for logits whose
// exponential is 0 too.  A NaN stays one (fmin and fmax would take the other operand).
static __device__ __forceinline__ void share(float logit, int m, double min_logit, const double2 *inverse, float &new_logit,
                                             float &shrink) {
    if (isnan(logit)) {
        new_logit = shrink = logit;
        return;
    }
    if (logit < -40.0f) {
        new_logit = (float)fmax((double)logit - log((double)m), min_logit);
        shrink = 0.0f;
        return;
    }
    const double x = fmin((double)logit, 16.0), z = log1p(exp(-fabs(x)));
    const double y = (fmax(x, 0.0) + z) / (double)m, p = -expm1(-y);   // softplus / m = -log(1 - o) / m
    double term = 1.0, sum = 0.0, left = (double)m * p;
    for (int j = 1; j <= kRelTerms && j <= m; j++) {
        const double2 r = inverse[j];
        term *= left * r.x;                    // C(m, j) p^j
        left -= p;
        sum += (j & 1) ? term * r.y : -(term * r.y);
        if (term < 1e-18 * sum) break;
    }
    new_logit = (float)fmax(log(expm1(y)), min_logit);
    shrink = (float)(fmin(x, 0.0) - z - log(sum));
}

__global__ void __launch_bounds__(kRelThreads)
k_relocate_rows(int pairs, const int32_t *__restrict__ targets, const int32_t *__restrict__ sources,
                const int32_t *__restrict__ copies, const RelocatePair *__restrict__ in, double min_logit,
                RelocateSets a) {
    __shared__ float fresh[kRowPairs][4];      // new log-scales, new logit
    __shared__ int32_t rank[kRowPairs], to[kRowPairs], from[kRowPairs];
    __shared__ double2 inverse[kRelTerms + 1];
    const int tid = threadIdx.x, first = blockIdx.x * kRowPairs;
    if (tid >= 64 && tid <= 64 + kRelTerms) {
        const double j = tid > 64 ? (double)(tid - 64) : 1.0;
        inverse[tid - 64] = make_double2(1.0 / j, 1.0 / sqrt(j));
    }
    RelocatePair p = {0.0f, 0.0f, 0.0f, 0.0f, -1};
    int32_t s = 0, m = 0;
    if (tid < kRowPairs && first + tid < pairs) {
        p = in[first + tid];
        if (p.rank >= 0) {
            s = sources[first + tid];
            m = copies[s] + 1;
            to[tid] = targets[first + tid];
            from[tid] = s;
        }
    }
    __syncthreads();
    if (tid < kRowPairs) {
        rank[tid] = p.rank;
        if (p.rank >= 0) {
            float l, d;
            share(p.logit, m, min_logit, inverse, l, d);
            fresh[tid][0] = p.s0 + d;
            fresh[tid][1] = p.s1 + d;
            fresh[tid][2] = p.s2 + d;
            fresh[tid][3] = l;
        }
    }
    __syncthreads();
    const int lane = tid & 63, k0 = (tid >> 6) * (kRowPairs / 4);
    for (int c0 = 0; c0 < a.columns; c0 += 64) {
        const int c = c0 + lane;
        if (c >= a.columns) continue;
        // the lane's tensor, its row length and the column in it
        float *tp = a.p[5], *tm = a.m[5], *tv = a.v[5];
        int len = a.columns - 14, off = c - 14, q = -1;   // q: the column of `fresh`
        if (c < 3) { tp = a.p[0]; tm = a.m[0]; tv = a.v[0]; len = 3; off = c; }
        else if (c < 6) { tp = a.p[1]; tm = a.m[1]; tv = a.v[1]; len = 3; off = q = c - 3; }
        else if (c < 10) { tp = a.p[2]; tm = a.m[2]; tv = a.v[2]; len = 4; off = c - 6; }
        else if (c < 11) { tp = a.p[3]; tm = a.m[3]; tv = a.v[3]; len = 1; off = 0; q = 3; }
        else if (c < 14) { tp = a.p[4]; tm = a.m[4]; tv = a.v[4]; len = 3; off = c - 11; }
        float v[kRowPairs / 4];
#pragma unroll
        for (int k = 0; k < kRowPairs / 4; k++) {
            v[k] = 0.0f;
            if (rank[k0 + k] >= 0) v[k] = q >= 0 ? fresh[k0 + k][q] : tp[(size_t)from[k0 + k] * len + off];
        }
#pragma unroll
        for (int k = 0; k < kRowPairs / 4; k++) {
            const int32_t rk = rank[k0 + k];
            if (rk < 0) continue;
            const size_t t = (size_t)to[k0 + k] * len + off, f = (size_t)from[k0 + k] * len + off;
            tp[t] = v[k];
            if (tm) tm[t] = 0.0f;
            if (tv) tv[t] = 0.0f;
            if (rk == 0) {
                if (q >= 0) tp[f] = v[k];
                if (tm) tm[f] = 0.0f;
                if (tv) tv[f] = 0.0f;
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
    if (pairs > 0x0fffffff) return GS_ERR_UNSUPPORTED;   // (a launch's threads, 32 bits)
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
    if (pairs <= kFewPairs) {
        GS_LAUNCH(k_relocate_few, dim3(1), dim3(kFewPairs), 0, s, N, pairs, targets, sources, owner, copies, p.opacity_logits,
                  p.log_scales, held);
        GS_LAUNCH_CHECK();
    } else {
        GS_LAUNCH(k_relocate_clear, grid, block, 0, s, N, pairs, targets, sources, owner, copies);
        GS_LAUNCH_CHECK();
        GS_LAUNCH(k_relocate_claim, grid, block, 0, s, N, pairs, targets, sources, owner);
        GS_LAUNCH_CHECK();
        GS_LAUNCH(k_relocate_count, grid, block, 0, s, N, pairs, targets, sources, owner, copies, p.opacity_logits,
                  p.log_scales, held);
        GS_LAUNCH_CHECK();
    }
    RelocateSets a = {{p.means, p.log_scales, p.quats, p.opacity_logits, p.features_dc, p.features_rest},
                      {m.means, m.log_scales, m.quats, m.opacity_logits, m.features_dc, m.features_rest},
                      {v.means, v.log_scales, v.quats, v.opacity_logits, v.features_dc, v.features_rest},
                      14 + (K - 1) * 3};
    const double o = (double)min_opacity;
    GS_LAUNCH(k_relocate_rows, dim3((pairs + kRowPairs - 1) / kRowPairs), block, 0, s, pairs, targets, sources, copies, held,
              log(o / (1.0 - o)), a);
    GS_LAUNCH_CHECK();
    return GS_OK;
}
