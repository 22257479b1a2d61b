// gs_sample.hip — indices drawn from given random numbers: rows of logits (or opacity logits), temperature, top-k,
// top-p, min-p.  C ABI: include/gsplat_densify.h (gs_sample), which also holds the definition.
//
//   order   entries by descending value, equal ones by ascending index; NaN and -inf are no candidates
//   weight  w = exp((l - max l) / T), l = x, or log sigmoid(x) for opacity logits
//   kept    the first k of the order; of these the shortest prefix whose mass reaches p times theirs; of these w >= min_p
//   draw    the lowest index whose running sum of kept weights, in index order, exceeds u times the total
//
// The kept entries are a prefix of the order up to min_p, so a row's selection is two numbers: a threshold key and how
// many of the entries that equal it are kept (the lowest indices).  Keys are the 32 bits of the value mapped so that
// unsigned order is value order; 0 stands for "no candidate".
//
// Weights and their sums are 64-bit: an index is right or wrong, and with 5 million candidates and 250 000 draws a
// 24-bit weight would move a border across a draw several times in every call.  Every sum has a fixed order.
#include <math.h>

#include "gs_device.h"
#include "../../include/gsplat_densify.h"

namespace gs {

constexpr int kSeg = 16;                       // entries one thread sums: the grain of the stored running sums
constexpr int kSelThreads = 1024;
constexpr int kSelChunk = kSelThreads * kSeg;  // entries a workgroup sums in one step

enum SampleDtype { kF32 = GS_DTYPE_F32, kF16 = GS_DTYPE_F16, kBF16 = GS_DTYPE_BF16 };

struct SampleArgs {
    const void *logits;
    int64_t stride;
    int rows, cols, draws;
    GsSampleConfig cfg;
};

// What the draws of a row need of its selection.
struct SampleRow {
    double total, inv_t, l_max, min_p;
    uint32_t max_key, threshold, ties;         // kept: key > threshold, and the first `ties` entries with key == threshold
    uint32_t pad;
};

// A row's settings; `ok` false: the row draws nothing.
struct RowSettings {
    double temperature, top_p, min_p;
    int64_t top_k;
    bool ok;
};

static __device__ __forceinline__ RowSettings row_settings(const SampleArgs &a, int r) {
    const GsSampleConfig &c = a.cfg;
    const float t = c.temperature_rows ? c.temperature_rows[r] : c.temperature;
    const float p = c.top_p_rows ? c.top_p_rows[r] : c.top_p;
    const float m = c.min_p_rows ? c.min_p_rows[r] : c.min_p;
    int64_t k = c.top_k_rows ? c.top_k_rows[r] : c.top_k;
    RowSettings s;
    s.ok = t >= 0.0f && !isnan(p) && !isnan(m);
    if (k <= 0) k = a.cols;
    // temperature 0, a min_p that nothing reaches, a top_p that asks for no mass: the first of the order alone
    if (t == 0.0f || m > 1.0f || p <= 0.0f) k = 1;
    s.top_k = k;
    s.temperature = t == 0.0f ? 1.0 : (double)t;
    s.top_p = (p < 1.0f && p > 0.0f) ? (double)p : 1.0;
    s.min_p = m > 1.0f ? 0.0 : (double)m;
    return s;
}

static __device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0u;           // NaN, -inf
    const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 and 0 are equal values)
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
static __device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

template <int DT>
static __device__ __forceinline__ float load_value(const void *row, int64_t i) {
    if constexpr (DT == kF32) return static_cast<const float *>(row)[i];
    if constexpr (DT == kBF16) return __uint_as_float((uint32_t)static_cast<const uint16_t *>(row)[i] << 16);
    return (float)static_cast<const _Float16 *>(row)[i];
}

template <bool OPACITY>
static __device__ __forceinline__ double log_weight(double x) {
    if constexpr (!OPACITY) return x;
    return x < 0.0 ? x - log1p(exp(x)) : -log1p(exp(-x));
}

template <bool OPACITY>
static __device__ __forceinline__ double weight(uint32_t key, const SampleRow &s) {
    if (key == s.max_key) return 1.0;          // (+inf - +inf)
    return exp((log_weight<OPACITY>((double)value_of(key)) - s.l_max) * s.inv_t);
}

// ---- workgroup sums, 1024 threads; every thread gets the result; fixed order ------------------------------------
static __device__ __forceinline__ double block_sum_d(double v, double *red /* [16] */) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = 0.0;
    for (int w = 0; w < kSelThreads / 64; w++) r += red[w];
    return r;
}
static __device__ __forceinline__ int64_t block_sum_i(int64_t v, double *red) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __longlong_as_double(v);
    __syncthreads();
    int64_t r = 0;
    for (int w = 0; w < kSelThreads / 64; w++) r += __double_as_longlong(red[w]);
    return r;
}

// One workgroup per row: maximum, threshold by bisection over the key's bits, running sums per 16 entries.
template <int DT, bool OPACITY>
__global__ void __launch_bounds__(kSelThreads)
k_sample_row(SampleArgs a, SampleRow *__restrict__ rows, double *__restrict__ seg_sum,
             uint32_t *__restrict__ seg_ties) {
    __shared__ double red[kSelThreads / 64];
    __shared__ double wave_sum[kSelThreads / 64];
    __shared__ uint32_t wave_tie[kSelThreads / 64];
    const int r = blockIdx.x, tid = threadIdx.x, n = a.cols;
    const char *row = static_cast<const char *>(a.logits) + (size_t)r * a.stride * (DT == kF32 ? 4 : 2);
    const RowSettings set = row_settings(a, r);
    auto key_at = [&](int64_t i) { return key_of(load_value<DT>(row, i)); };

    uint32_t mx = 0;
    for (int64_t i = tid; i < n; i += kSelThreads) mx = max(mx, key_at(i));
    for (int off = 32; off > 0; off >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, off, 64));
    if ((tid & 63) == 0) wave_tie[tid >> 6] = mx;
    __syncthreads();
    for (int w = 0; w < kSelThreads / 64; w++) mx = max(mx, wave_tie[w]);
    __syncthreads();

    SampleRow s;
    s.max_key = mx;
    s.inv_t = 1.0 / set.temperature;
    s.l_max = log_weight<OPACITY>((double)value_of(mx));
    s.min_p = set.min_p;
    s.threshold = 0;
    s.ties = 0;
    s.total = 0.0;
    s.pad = 0;
    const bool any = set.ok && mx != 0;
    auto count_from = [&](uint32_t t) {
        int64_t c = 0;
        for (int64_t i = tid; i < n; i += kSelThreads) c += key_at(i) >= t;
        return block_sum_i(c, red);
    };
    auto mass_from = [&](uint32_t t) {
        double m = 0.0;
        for (int64_t i = tid; i < n; i += kSelThreads) {
            const uint32_t k = key_at(i);
            if (k >= t) m += weight<OPACITY>(k, s);
        }
        return block_sum_d(m, red);
    };
    if (any && set.top_k < n && count_from(1u) > set.top_k) {
        uint32_t t = 0;                        // largest key with at least top_k entries from it on
        for (int b = 31; b >= 0; b--)
            if (count_from(t | (1u << b)) >= set.top_k) t |= 1u << b;
        s.threshold = t;
        s.ties = (uint32_t)(set.top_k - (t == 0xFFFFFFFFu ? 0 : count_from(t + 1u)));
    }
    if (any && set.top_p < 1.0) {
        const uint32_t kt = s.threshold;
        const double tie_mass = kt ? (double)s.ties * weight<OPACITY>(kt, s) : 0.0;
        const double goal = set.top_p * (mass_from(kt + 1u) + tie_mass);
        uint32_t t = 0;                        // largest key with mass >= goal from it on, inside the first k
        for (int b = 31; b >= 0; b--) {
            const uint32_t c = t | (1u << b);
            if (c <= kt || mass_from(c) >= goal) t = c;
        }
        if (t > kt) {
            const double above = t == 0xFFFFFFFFu ? 0.0 : mass_from(t + 1u), w = weight<OPACITY>(t, s);
            const int64_t have = count_from(t) - (t == 0xFFFFFFFFu ? 0 : count_from(t + 1u));
            int64_t c = w > 0.0 ? (int64_t)fmin(ceil((goal - above) / w), (double)have) : have;
            s.threshold = t;
            s.ties = (uint32_t)max(c, (int64_t)1);
        } else if (kt) {                       // the border lies among the ties that top-k left
            const double above = mass_from(kt + 1u), w = weight<OPACITY>(kt, s);
            const double c = w > 0.0 ? ceil((goal - above) / w) : (double)s.ties;
            s.ties = (uint32_t)fmin(fmax(c, 1.0), (double)s.ties);
        }
    }

    // running sums in index order
    double base = 0.0;
    uint32_t tie_base = 0;
    const int64_t nseg = (n + kSeg - 1) / kSeg;
    double *out_sum = seg_sum + (size_t)r * nseg;
    uint32_t *out_tie = seg_ties + (size_t)r * nseg;
    for (int64_t first = 0; any && first < n; first += kSelChunk) {
        const int64_t i0 = first + (int64_t)tid * kSeg, i1 = min(i0 + kSeg, (int64_t)n);
        uint32_t tie = 0;
        for (int64_t i = i0; i < i1; i++) tie += s.threshold != 0 && key_at(i) == s.threshold;
        // exclusive scans over the workgroup: ties first, they decide what the sums hold
        uint32_t ti = tie;
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)ti, off, 64);
            if ((tid & 63) >= off) ti += o;
        }
        __syncthreads();
        if ((tid & 63) == 63) wave_tie[tid >> 6] = ti;
        __syncthreads();
        uint32_t before = tie_base + ti - tie, all_ties = 0;
        for (int w = 0; w < kSelThreads / 64; w++) {
            if (w < (tid >> 6)) before += wave_tie[w];
            all_ties += wave_tie[w];
        }
        double sum = 0.0;
        uint32_t rank = before;
        for (int64_t i = i0; i < i1; i++) {
            const uint32_t k = key_at(i);
            const bool tied = s.threshold != 0 && k == s.threshold;
            const bool kept = k > s.threshold || (tied && rank < s.ties);
            rank += tied;
            if (!kept) continue;
            const double w = weight<OPACITY>(k, s);
            if (w >= s.min_p) sum += w;
        }
        double inc = sum;
        for (int off = 1; off < 64; off <<= 1) {
            const double o = __shfl_up(inc, off, 64);
            if ((tid & 63) >= off) inc += o;
        }
        __syncthreads();
        if ((tid & 63) == 63) wave_sum[tid >> 6] = inc;
        __syncthreads();
        double pre = 0.0, chunk = 0.0;
        for (int w = 0; w < kSelThreads / 64; w++) {
            if (w == (tid >> 6)) pre = chunk;
            chunk += wave_sum[w];
        }
        if (i0 < n) {
            const double excl = __shfl_up(inc, 1, 64);
            out_sum[i0 / kSeg] = base + (pre + ((tid & 63) ? excl : 0.0));
            out_tie[i0 / kSeg] = before;
        }
        base += chunk;
        tie_base += all_ties;
    }
    s.total = any ? base : 0.0;
    if (tid == 0) rows[r] = s;
}

// One thread per draw: the last segment whose running sum does not exceed the goal, then its entries one by one.
template <int DT, bool OPACITY>
__global__ void __launch_bounds__(256)
k_sample_draw(SampleArgs a, const SampleRow *__restrict__ rows, const double *__restrict__ seg_sum,
              const uint32_t *__restrict__ seg_ties, const float *__restrict__ uniforms, int32_t *__restrict__ ids) {
    const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= (int64_t)a.rows * a.draws) return;
    const int r = (int)(at / a.draws), n = a.cols;
    const SampleRow s = rows[r];
    const float u = uniforms[at];
    if (!(s.total > 0.0) || isnan(u)) {
        ids[at] = -1;
        return;
    }
    double goal = (double)u * s.total;
    if (goal < 0.0) goal = 0.0;
    if (goal >= s.total) goal = s.total * (1.0 - 0x1p-53);
    const int64_t nseg = ((int64_t)n + kSeg - 1) / kSeg;
    const double *sums = seg_sum + (size_t)r * nseg;
    int64_t lo = 0, hi = nseg;                 // sums[lo] <= goal < sums[hi]
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (sums[mid] <= goal) lo = mid;
        else hi = mid;
    }
    const char *row = static_cast<const char *>(a.logits) + (size_t)r * a.stride * (DT == kF32 ? 4 : 2);
    double c = sums[lo];
    uint32_t rank = seg_ties[(size_t)r * nseg + lo];
    int64_t id = -1;
    const int64_t i1 = min((lo + 1) * kSeg, (int64_t)n);
    for (int64_t i = lo * kSeg; i < i1; i++) {
        const uint32_t k = key_of(load_value<DT>(row, i));
        const bool tied = s.threshold != 0 && k == s.threshold;
        const bool kept = k > s.threshold || (tied && rank < s.ties);
        rank += tied;
        if (!kept) continue;
        const double w = weight<OPACITY>(k, s);
        if (!(w >= s.min_p) || !(w > 0.0)) continue;
        c += w;
        id = i;                                // (rounding of the last sum: the last entry that can be drawn)
        if (c > goal) break;
    }
    ids[at] = (int32_t)id;
}

struct SampleLayout {
    size_t rows_off, sum_off, tie_off, total;
    SampleLayout(int rows, int cols) {
        size_t o = 0;
        auto take = [&](size_t bytes) { size_t r = o; o += (bytes + 255) & ~(size_t)255; return r; };
        const size_t nseg = ((size_t)cols + kSeg - 1) / kSeg;
        rows_off = take((size_t)rows * sizeof(SampleRow));
        sum_off = take((size_t)rows * nseg * sizeof(double));
        tie_off = take((size_t)rows * nseg * sizeof(uint32_t));
        total = o;
    }
};

template <int DT, bool OPACITY>
static int launch_sample(const SampleArgs &a, const float *uniforms, int32_t *ids, char *ws, const SampleLayout &L,
                         hipStream_t s) {
    SampleRow *rows = (SampleRow *)(ws + L.rows_off);
    double *sums = (double *)(ws + L.sum_off);
    uint32_t *ties = (uint32_t *)(ws + L.tie_off);
    GS_LAUNCH((k_sample_row<DT, OPACITY>), dim3(a.rows), dim3(kSelThreads), 0, s, a, rows, sums, ties);
    GS_LAUNCH_CHECK();
    const int64_t want = ((int64_t)a.rows * a.draws + 255) / 256;
    GS_LAUNCH((k_sample_draw<DT, OPACITY>), dim3((unsigned)want), dim3(256), 0, s, a, rows, sums, ties, uniforms, ids);
    GS_LAUNCH_CHECK();
    return GS_OK;
}

}  // namespace gs

extern "C" size_t gs_sample_workspace_bytes(int rows, int cols) {
    if (rows <= 0 || cols < 0) return 0;
    return gs::SampleLayout(rows, cols).total;
}

extern "C" int gs_sample(int rows, int cols, const void *logits, int64_t row_stride, const GsSampleConfig *cfg, int draws,
                         const float *uniforms, int32_t *ids, void *workspace, size_t workspace_bytes,
                         gs_stream_t stream) {
    using namespace gs;
    if (rows < 0 || cols < 0 || draws < 0 || !cfg) return GS_ERR_INVALID_ARGUMENT;
    if (cfg->dtype != kF32 && cfg->dtype != kF16 && cfg->dtype != kBF16) return GS_ERR_INVALID_ARGUMENT;
    if (cfg->flags & ~(uint32_t)GS_FLAG_LOGIT_OPACITY) return GS_ERR_INVALID_ARGUMENT;
    if (!(cfg->temperature >= 0.0f) || isnan(cfg->top_p) || !(cfg->min_p <= 1.0f)) return GS_ERR_INVALID_ARGUMENT;
    if (rows == 0 || draws == 0) return GS_OK;
    if ((cols > 0 && !logits) || !uniforms || !ids || !workspace) return GS_ERR_INVALID_ARGUMENT;
    if (rows > 1 && row_stride < cols) return GS_ERR_INVALID_ARGUMENT;
    const size_t size = cfg->dtype == kF32 ? 4 : 2;
    if (((uintptr_t)logits & (size - 1)) || ((uintptr_t)workspace & 15) || (((uintptr_t)uniforms | (uintptr_t)ids) & 3))
        return GS_ERR_INVALID_ARGUMENT;
    if ((int64_t)rows * draws > 0x7fffffffLL * 128) return GS_ERR_INVALID_ARGUMENT;
    const SampleLayout L(rows, cols);
    if (workspace_bytes < L.total) return GS_ERR_WORKSPACE;
    SampleArgs a = {logits, row_stride, rows, cols, draws, *cfg};
    const bool op = cfg->flags & GS_FLAG_LOGIT_OPACITY;
    hipStream_t s = (hipStream_t)stream;
    char *ws = (char *)workspace;
    switch (cfg->dtype) {
    case kF32: return op ? launch_sample<kF32, true>(a, uniforms, ids, ws, L, s)
                         : launch_sample<kF32, false>(a, uniforms, ids, ws, L, s);
    case kF16: return op ? launch_sample<kF16, true>(a, uniforms, ids, ws, L, s)
                         : launch_sample<kF16, false>(a, uniforms, ids, ws, L, s);
    default: return op ? launch_sample<kBF16, true>(a, uniforms, ids, ws, L, s)
                       : launch_sample<kBF16, false>(a, uniforms, ids, ws, L, s);
    }
}
