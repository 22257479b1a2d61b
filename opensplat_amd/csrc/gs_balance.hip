// gs_balance.hip — the balance loss of a frame's tile lists with its gradient.  C ABI: include/gsplat_train.h
// (gs_tile_balance), which also holds the definition.
//
//   loss = T / (M S) sum_t n_t S_t,   n_t entries of tile t, S_t the opacity in its list, M and S their sums over T tiles
//
// Exchanging the sums, sum_t n_t S_t = sum_g o_g A_g with A_g = the entries of all the tiles that Gaussian g's rectangle
// covers — and over a rectangle of tiles that is four look-ups in a summed-area table of the n_t.  No list is walked:
// the lists' 4 bytes per entry, their opacities and a gradient scattered back through them fall away, and what remains
// is one pass over the records.
//
//   k_balance_sums   the table, by every workgroup for itself in LDS (up to 38 k tiles, 4K frames); per Gaussian A_g, c_g and
//                    o_g, kept for the next launch, and sum o_g A_g, sum o_g c_g per workgroup in 64 bits
//   k_balance_grad   the loss, and d loss / d o_g = T / (M S) (A_g - c_g Q / S), Q = sum o A
// Larger frames: k_balance_rows and k_balance_cols leave the table in memory.
//
// Bound by the records' lines: 12 of a record's 48 bytes are used and no line is without some, 240 MB at 5 M Gaussians.
// The second launch reads the 12 bytes kept (60 MB) instead of the records again.  Measured: 1 M Gaussians at 1080p 19 + 6
// us, 5 M at 4K 74 + 14 us (4.1 TB/s in the first launch, a large copy reaches 4.9; 5 us of it before the table is made).
// With the table from memory and the records read twice it was 48 and 164 us.
#include <math.h>

#include "gs_device.h"
#include "../../include/gsplat_train.h"

namespace gs {

constexpr int kBalThreads = 256;

struct BalanceGrid {
    int tw, th, pitch;                         // tiles across and down; entries per row of the table
};

__global__ void __launch_bounds__(kBalThreads)
k_balance_rows(BalanceGrid g, const int2 *__restrict__ bins, int32_t *__restrict__ counts, int32_t *__restrict__ table) {
    __shared__ int32_t wave_sum[kBalThreads / 64];
    const int y = blockIdx.x, tid = threadIdx.x;
    int32_t *out = table + (size_t)(y + 1) * g.pitch;
    if (tid == 0) out[0] = 0;
    if (y == 0)
        for (int x = tid; x < g.pitch; x += kBalThreads) table[x] = 0;
    int32_t base = 0;
    for (int x0 = 0; x0 < g.tw; x0 += kBalThreads) {
        const int x = x0 + tid;
        int32_t n = 0;
        if (x < g.tw) {
            const int2 b = bins[(size_t)y * g.tw + x];
            n = b.y - b.x;
            if (counts) counts[(size_t)y * g.tw + x] = n;
        }
        int32_t s = n;
        for (int off = 1; off < 64; off <<= 1) {
            const int32_t o = __shfl_up(s, off, 64);
            if ((tid & 63) >= off) s += o;
        }
        __syncthreads();
        if ((tid & 63) == 63) wave_sum[tid >> 6] = s;
        __syncthreads();
        int32_t pre = base;
        for (int w = 0; w < kBalThreads / 64; w++) {
            if (w < (tid >> 6)) pre += wave_sum[w];
            base += wave_sum[w];
        }
        if (x < g.tw) out[x + 1] = pre + s;
    }
}

// Down the columns, a thread each, eight rows' loads under way together.
__global__ void __launch_bounds__(64)
k_balance_cols(BalanceGrid g, int32_t *__restrict__ table) {
    const int x = blockIdx.x * 64 + threadIdx.x;
    if (x >= g.pitch) return;
    int32_t s = 0;
    for (int y = 1; y <= g.th; y += 8) {
        int32_t v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = y + k <= g.th ? table[(size_t)(y + k) * g.pitch + x] : 0;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            s += v[k];
            if (y + k <= g.th) table[(size_t)(y + k) * g.pitch + x] = s;
        }
    }
}

// Covered tiles of a record and the entries they hold.  (Coordinates clamped to the frame: a record of another frame
// reads no memory outside the table.)
struct Cover {
    int32_t tiles;
    int32_t entries;
};
static __device__ __forceinline__ Cover cover_of(const BalanceGrid &g, const int32_t *table, uint32_t rx, uint32_t ry) {
    const int x0 = (int)(rx & 0xFFFFu), x1 = (int)(rx >> 16), y0 = (int)(ry & 0xFFFFu), y1 = (int)(ry >> 16);
    if (x1 <= x0 || y1 <= y0) return {0, 0};
    const int a = min(x0 / GS_TILE, g.tw), b = min((x1 + GS_TILE - 1) / GS_TILE, g.tw);
    const int c = min(y0 / GS_TILE, g.th), d = min((y1 + GS_TILE - 1) / GS_TILE, g.th);
    const int32_t *top = table + (size_t)c * g.pitch, *bot = table + (size_t)d * g.pitch;
    return {(b - a) * (d - c), (bot[b] - top[b]) - (bot[a] - top[a])};
}

template <int THREADS>
static __device__ __forceinline__ double block_sum_f64(double v, double *red /* LDS [THREADS / 64] */) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) r += red[w];
    return r;
}

constexpr int kSumThreads = 1024;
constexpr int kSumParts = 256;                 // workgroups at most: one per compute unit
constexpr int kColParts = 4;

// The summed-area table of the lists' lengths in LDS.  A wave scans a tile row; a column is scanned in four parts, whose
// totals are added to the parts below it.
static __device__ __forceinline__ void lds_table(const BalanceGrid &g, const int2 *__restrict__ bins,
                                                 int32_t *__restrict__ counts, int32_t *table, int32_t *part_sum) {
    const int tid = threadIdx.x, lane = tid & 63, tiles = g.tw * g.th;
    for (int i0 = 0; i0 < tiles; i0 += 8 * kSumThreads) {
        int32_t n[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int i = i0 + k * kSumThreads + tid;
            n[k] = 0;
            if (i < tiles) {
                const int2 b = bins[i];
                n[k] = b.y - b.x;
            }
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int i = i0 + k * kSumThreads + tid;
            if (i < tiles) {
                const int y = i / g.tw, x = i - y * g.tw;
                table[(y + 1) * g.pitch + x + 1] = n[k];
                if (counts) counts[i] = n[k];
            }
        }
    }
    for (int x = tid; x < g.pitch; x += kSumThreads) table[x] = 0;
    for (int y = tid; y < g.th; y += kSumThreads) table[(y + 1) * g.pitch] = 0;
    __syncthreads();
    for (int y = 1 + (tid >> 6); y <= g.th; y += kSumThreads / 64) {
        int32_t base = 0;
        for (int x0 = 1; x0 <= g.tw; x0 += 64) {
            const int x = x0 + lane;
            const int32_t s = (int32_t)wave_scan((uint32_t)(x <= g.tw ? table[y * g.pitch + x] : 0));
            if (x <= g.tw) table[y * g.pitch + x] = base + s;
            base += __builtin_amdgcn_readlane(s, 63);
        }
    }
    __syncthreads();
    const int part_rows = (g.th + kColParts - 1) / kColParts;
    constexpr int kCols = kSumThreads / kColParts;
    const int part = tid / kCols, y0 = 1 + part * part_rows, y1 = min(y0 + part_rows, g.th + 1);
    for (int x0 = 0; x0 < g.pitch; x0 += kCols) {
        const int x = x0 + (tid & (kCols - 1));
        int32_t s = 0;
        if (x < g.pitch)
#pragma unroll 8
            for (int y = y0; y < y1; y++) s += table[y * g.pitch + x];
        part_sum[tid] = s;
        __syncthreads();
        s = 0;
        for (int p = 0; p < part; p++) s += part_sum[p * kCols + (tid & (kCols - 1))];
        if (x < g.pitch)
#pragma unroll 8
            for (int y = y0; y < y1; y++) {
                s += table[y * g.pitch + x];
                table[y * g.pitch + x] = s;
            }
        __syncthreads();
    }
}

template <bool LDS>
__global__ void __launch_bounds__(kSumThreads)
k_balance_sums(BalanceGrid g, int N, const float *__restrict__ packed, const int2 *__restrict__ bins,
               int32_t *__restrict__ counts, const int32_t *__restrict__ table_mem, int2 *__restrict__ cover,
               float *__restrict__ opacity, double2 *__restrict__ parts, int32_t *__restrict__ entries) {
    __shared__ double red[kSumThreads / 64];
    __shared__ int32_t part_sum[kSumThreads];
    extern __shared__ int32_t table_lds[];
    // Four records a thread are under way at a time: the first while the table is made, the next while these are looked up.
    struct Batch {
        float o[4];
        uint32_t rx[4], ry[4];
    };
    const int64_t stride = (int64_t)gridDim.x * kSumThreads;
    auto load = [&](int64_t n0) {
        Batch b;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t n = n0 + k * stride;
            b.rx[k] = b.ry[k] = 0;
            b.o[k] = 0.0f;
            if (n < N) {
                const float *p = packed + (size_t)n * GS_SPLAT_DWORDS;
                b.o[k] = p[5];
                b.rx[k] = __float_as_uint(p[7]);
                b.ry[k] = __float_as_uint(p[11]);
            }
        }
        return b;
    };
    int64_t n0 = (int64_t)blockIdx.x * kSumThreads + threadIdx.x;
    Batch next = load(n0);
    const int32_t *table = table_mem;
    if constexpr (LDS) {
        lds_table(g, bins, blockIdx.x == 0 ? counts : nullptr, table_lds, part_sum);
        table = table_lds;
    }
    double q = 0.0, s = 0.0;
    for (; n0 < N; n0 += 4 * stride) {
        const Batch b = next;
        next = load(n0 + 4 * stride);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t n = n0 + k * stride;
            if (n >= N) continue;
            const Cover c = cover_of(g, table, b.rx[k], b.ry[k]);
            cover[n] = make_int2(c.entries, c.tiles);
            opacity[n] = b.o[k];
            if (c.tiles > 0) {
                q += (double)b.o[k] * (double)c.entries;
                s += (double)b.o[k] * (double)c.tiles;
            }
        }
    }
    q = block_sum_f64<kSumThreads>(q, red);
    s = block_sum_f64<kSumThreads>(s, red);
    if (threadIdx.x == 0) {
        parts[blockIdx.x] = make_double2(q, s);
        if (blockIdx.x == 0) *entries = table[(size_t)g.th * g.pitch + g.tw];
    }
}

__global__ void __launch_bounds__(kBalThreads)
k_balance_grad(BalanceGrid g, int N, int nparts, const double2 *__restrict__ parts, const int32_t *__restrict__ entries,
               const int2 *__restrict__ cover, const float *__restrict__ opacity, double scale, uint32_t flags,
               float *__restrict__ loss, float *__restrict__ v_opacity) {
    __shared__ double red[kBalThreads / 64];
    double q = 0.0, s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += kBalThreads) {
        q += parts[i].x;
        s += parts[i].y;
    }
    q = block_sum_f64<kBalThreads>(q, red);
    s = block_sum_f64<kBalThreads>(s, red);
    const double m = (double)*entries;
    const bool some = m > 0.0 && s != 0.0;     // (a NaN among the opacities shows in all that depends on it)
    const double norm = some ? (double)g.tw * (double)g.th / m : 0.0, mean = some ? q / s : 0.0;
    if (blockIdx.x == 0 && threadIdx.x == 0) loss[0] = (float)(scale * (norm * mean));
    if (!v_opacity) return;
    const double k = some ? scale * norm / s : 0.0;
    auto slope = [&](int entries_, int tiles, float op) {
        if (!some || tiles <= 0) return 0.0f;
        double v = k * ((double)entries_ - (double)tiles * mean);
        if (flags & GS_FLAG_LOGIT_OPACITY) v *= (double)op * (1.0 - (double)op);
        return (float)v;
    };
    const bool add = flags & GS_FLAG_ACCUMULATE_GRADS;
    const int64_t step = (int64_t)gridDim.x * kBalThreads * 4;
    for (int64_t n = ((int64_t)blockIdx.x * kBalThreads + threadIdx.x) * 4; n < N; n += step) {
        // (the workspace's arrays are padded to whole fours; v_opacity may have any alignment of a float)
        const int4 c0 = *reinterpret_cast<const int4 *>(cover + n), c1 = *reinterpret_cast<const int4 *>(cover + n + 2);
        const float4 op = *reinterpret_cast<const float4 *>(opacity + n);
        const float v[4] = {slope(c0.x, c0.y, op.x), slope(c0.z, c0.w, op.y), slope(c1.x, c1.y, op.z), slope(c1.z, c1.w, op.w)};
        const bool in[4] = {c0.y > 0, c0.w > 0, c1.y > 0, c1.w > 0};
        if (!add && n + 4 <= N) {
            __builtin_memcpy(v_opacity + n, v, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (n + e >= N) break;
                if (!add) v_opacity[n + e] = v[e];
                else if (in[e]) v_opacity[n + e] += v[e];
            }
        }
    }
}

// Tables up to here fit in the 160 KB of LDS beside the workgroup's own 4.2 KB (38 400 tiles; 4K frames have 32 400).
constexpr size_t kLdsTable = 150 * 1024;

struct BalanceLayout {
    BalanceGrid g;
    size_t table_bytes, table, parts, entries, cover, opacity, total;
    bool lds;
    BalanceLayout(int W, int H, int N) {
        g.tw = (W + GS_TILE - 1) / GS_TILE;
        g.th = (H + GS_TILE - 1) / GS_TILE;
        g.pitch = g.tw + 1;
        table_bytes = (size_t)g.pitch * (g.th + 1) * sizeof(int32_t);
        lds = table_bytes <= kLdsTable;
        size_t o = 0;
        auto take = [&](size_t bytes) { size_t r = o; o += (bytes + 255) & ~(size_t)255; return r; };
        table = take(lds ? 0 : table_bytes);
        parts = take((size_t)kSumParts * sizeof(double2));
        entries = take(sizeof(int32_t));
        cover = take(((size_t)N + 3) * sizeof(int2));
        opacity = take(((size_t)N + 3) * sizeof(float));
        total = o;
    }
};

}  // namespace gs

extern "C" size_t gs_tile_balance_workspace_bytes(int W, int H, int N) {
    if (W <= 0 || H <= 0 || W > 65535 || H > 65535 || N < 0) return 0;
    return gs::BalanceLayout(W, H, N).total;
}

extern "C" int gs_tile_balance(int W, int H, int N, const float *packed, const int32_t *tile_bins, float scale,
                               float *loss, int32_t *counts, float *v_opacity, uint32_t flags, void *workspace,
                               size_t workspace_bytes, gs_stream_t stream) {
    using namespace gs;
    if (W <= 0 || H <= 0 || N < 0 || !tile_bins || !loss || !workspace) return GS_ERR_INVALID_ARGUMENT;
    if (W > 65535 || H > 65535) return GS_ERR_UNSUPPORTED;
    if (N > 0 && !packed) return GS_ERR_INVALID_ARGUMENT;
    if (flags & ~(uint32_t)(GS_FLAG_LOGIT_OPACITY | GS_FLAG_ACCUMULATE_GRADS)) return GS_ERR_INVALID_ARGUMENT;
    if (!(scale >= -3.0e38f && scale <= 3.0e38f)) return GS_ERR_INVALID_ARGUMENT;
    if ((flags & GS_FLAG_ACCUMULATE_GRADS) && !v_opacity) return GS_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)packed & 15) || ((uintptr_t)tile_bins & 7) || ((uintptr_t)workspace & 15) ||
        (((uintptr_t)loss | (uintptr_t)counts | (uintptr_t)v_opacity) & 3))
        return GS_ERR_INVALID_ARGUMENT;
    const BalanceLayout L(W, H, N);
    if (workspace_bytes < L.total) return GS_ERR_WORKSPACE;
    char *ws = (char *)workspace;
    int32_t *table = (int32_t *)(ws + L.table), *entries = (int32_t *)(ws + L.entries);
    double2 *parts = (double2 *)(ws + L.parts);
    int2 *cover = (int2 *)(ws + L.cover);
    float *opacity = (float *)(ws + L.opacity);
    hipStream_t s = (hipStream_t)stream;
    const int2 *bins = (const int2 *)tile_bins;
    // one Gaussian a thread at least
    const int64_t want = ((int64_t)N + kSumThreads - 1) / kSumThreads, most = kSumParts;
    const int blocks = (int)(want < 1 ? 1 : (want < most ? want : most));
    if (L.lds) {
        if (L.table_bytes > 48 * 1024)         // (beyond what every launch may have)
            GS_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(k_balance_sums<true>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLdsTable));
        GS_LAUNCH((k_balance_sums<true>), dim3(blocks), dim3(kSumThreads), L.table_bytes, s, L.g, N, packed, bins, counts,
                  (const int32_t *)nullptr, cover, opacity, parts, entries);
    } else {
        GS_LAUNCH(k_balance_rows, dim3(L.g.th), dim3(kBalThreads), 0, s, L.g, bins, counts, table);
        GS_LAUNCH_CHECK();
        GS_LAUNCH(k_balance_cols, dim3((L.g.pitch + 63) / 64), dim3(64), 0, s, L.g, table);
        GS_LAUNCH_CHECK();
        GS_LAUNCH((k_balance_sums<false>), dim3(blocks), dim3(kSumThreads), 0, s, L.g, N, packed, bins, counts, table, cover,
                  opacity, parts, entries);
    }
    GS_LAUNCH_CHECK();
    const int64_t grads = v_opacity ? ((int64_t)N + 4 * kBalThreads - 1) / (4 * kBalThreads) : 1;
    GS_LAUNCH(k_balance_grad, dim3((unsigned)(grads < 1 ? 1 : (grads < 1024 ? grads : 1024))), dim3(kBalThreads), 0, s, L.g, N,
              blocks, parts, entries, cover, opacity, (double)scale, flags, loss, v_opacity);
    GS_LAUNCH_CHECK();
    return GS_OK;
}
