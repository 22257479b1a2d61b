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
//   k_balance_rows   one workgroup per tile row: the counts, and their running sums along the row
//   k_balance_cols   one thread per tile column: down the rows
//   k_balance_sums   sum o_g A_g and sum o_g c_g (c_g covered tiles) per workgroup, in 64 bits
//   k_balance_grad   the loss, and d loss / d o_g = T / (M S) (A_g - c_g Q / S), Q = sum o A
#include <math.h>

#include "gs_device.h"
#include "../../include/gsplat_train.h"

namespace gs {

constexpr int kBalThreads = 256;
constexpr int kBalMaxParts = 1024;

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

__global__ void __launch_bounds__(64)
k_balance_cols(BalanceGrid g, int32_t *__restrict__ table) {
    const int x = blockIdx.x * 64 + threadIdx.x;
    if (x >= g.pitch) return;
    int32_t s = 0;
    for (int y = 1; y <= g.th; y++) {
        s += table[(size_t)y * g.pitch + x];
        table[(size_t)y * g.pitch + x] = s;
    }
}

// Covered tiles of a record and the entries they hold.  (Coordinates clamped to the frame: a record of another frame
// reads no memory outside the table.)
struct Cover {
    int32_t tiles;
    int32_t entries;
};
static __device__ __forceinline__ Cover cover_of(const BalanceGrid &g, const int32_t *__restrict__ table, uint32_t rx,
                                                 uint32_t ry) {
    const int x0 = (int)(rx & 0xFFFFu), x1 = (int)(rx >> 16), y0 = (int)(ry & 0xFFFFu), y1 = (int)(ry >> 16);
    if (x1 <= x0 || y1 <= y0) return {0, 0};
    const int a = min(x0 / GS_TILE, g.tw), b = min((x1 + GS_TILE - 1) / GS_TILE, g.tw);
    const int c = min(y0 / GS_TILE, g.th), d = min((y1 + GS_TILE - 1) / GS_TILE, g.th);
    const int32_t *top = table + (size_t)c * g.pitch, *bot = table + (size_t)d * g.pitch;
    return {(b - a) * (d - c), (bot[b] - top[b]) - (bot[a] - top[a])};
}

static __device__ __forceinline__ double block_sum_f64(double v, double *red) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ void __launch_bounds__(kBalThreads)
k_balance_sums(BalanceGrid g, int N, const float *__restrict__ packed, const int32_t *__restrict__ table,
               double2 *__restrict__ parts) {
    __shared__ double red[kBalThreads / 64];
    double q = 0.0, s = 0.0;
    for (int64_t n = (int64_t)blockIdx.x * kBalThreads + threadIdx.x; n < N; n += (int64_t)gridDim.x * kBalThreads) {
        const float *p = packed + (size_t)n * GS_SPLAT_DWORDS;
        const Cover c = cover_of(g, table, __float_as_uint(p[7]), __float_as_uint(p[11]));
        if (c.tiles > 0) {
            const double o = (double)p[5];
            q += o * (double)c.entries;
            s += o * (double)c.tiles;
        }
    }
    q = block_sum_f64(q, red);
    s = block_sum_f64(s, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = make_double2(q, s);
}

__global__ void __launch_bounds__(kBalThreads)
k_balance_grad(BalanceGrid g, int N, const float *__restrict__ packed, const int32_t *__restrict__ table, int nparts,
               const double2 *__restrict__ parts, double scale, uint32_t flags, float *__restrict__ loss,
               float *__restrict__ v_opacity) {
    __shared__ double red[kBalThreads / 64];
    double q = 0.0, s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += kBalThreads) {
        q += parts[i].x;
        s += parts[i].y;
    }
    q = block_sum_f64(q, red);
    s = block_sum_f64(s, red);
    const double entries = (double)table[(size_t)g.th * g.pitch + g.tw];
    const bool some = entries > 0.0 && s > 0.0;
    const double norm = some ? (double)g.tw * (double)g.th / entries : 0.0, mean = some ? q / s : 0.0;
    if (blockIdx.x == 0 && threadIdx.x == 0) loss[0] = (float)(scale * (norm * mean));
    if (!v_opacity) return;
    const double k = some ? scale * norm / s : 0.0;
    for (int64_t n = (int64_t)blockIdx.x * kBalThreads + threadIdx.x; n < N; n += (int64_t)gridDim.x * kBalThreads) {
        const float *p = packed + (size_t)n * GS_SPLAT_DWORDS;
        const Cover c = cover_of(g, table, __float_as_uint(p[7]), __float_as_uint(p[11]));
        double v = 0.0;
        if (some && c.tiles > 0) {
            v = k * ((double)c.entries - (double)c.tiles * mean);
            const double o = (double)p[5];
            if (flags & GS_FLAG_LOGIT_OPACITY) v *= o * (1.0 - o);
        }
        if (flags & GS_FLAG_ACCUMULATE_GRADS) {
            if (c.tiles > 0) v_opacity[n] += (float)v;
        } else {
            v_opacity[n] = (float)v;
        }
    }
}

struct BalanceLayout {
    BalanceGrid g;
    size_t table_off, parts_off, total;
    BalanceLayout(int W, int H) {
        g.tw = (W + GS_TILE - 1) / GS_TILE;
        g.th = (H + GS_TILE - 1) / GS_TILE;
        g.pitch = g.tw + 1;
        table_off = 0;
        parts_off = (((size_t)g.pitch * (g.th + 1) * sizeof(int32_t)) + 255) & ~(size_t)255;
        total = parts_off + (size_t)kBalMaxParts * sizeof(double2);
    }
};

}  // namespace gs

extern "C" size_t gs_tile_balance_workspace_bytes(int W, int H) {
    if (W <= 0 || H <= 0 || W > 65535 || H > 65535) return 0;
    return gs::BalanceLayout(W, H).total;
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
    const BalanceLayout L(W, H);
    if (workspace_bytes < L.total) return GS_ERR_WORKSPACE;
    char *ws = (char *)workspace;
    int32_t *table = (int32_t *)(ws + L.table_off);
    double2 *parts = (double2 *)(ws + L.parts_off);
    hipStream_t s = (hipStream_t)stream;
    const int64_t want = ((int64_t)N + kBalThreads - 1) / kBalThreads;
    const int blocks = (int)(want < 1 ? 1 : (want < kBalMaxParts ? want : kBalMaxParts));
    GS_LAUNCH(k_balance_rows, dim3(L.g.th), dim3(kBalThreads), 0, s, L.g, (const int2 *)tile_bins, counts, table);
    GS_LAUNCH_CHECK();
    GS_LAUNCH(k_balance_cols, dim3((L.g.pitch + 63) / 64), dim3(64), 0, s, L.g, table);
    GS_LAUNCH_CHECK();
    GS_LAUNCH(k_balance_sums, dim3(blocks), dim3(kBalThreads), 0, s, L.g, N, packed, table, parts);
    GS_LAUNCH_CHECK();
    GS_LAUNCH(k_balance_grad, dim3(blocks), dim3(kBalThreads), 0, s, L.g, N, packed, table, blocks, parts,
              (double)scale, flags, loss, v_opacity);
    GS_LAUNCH_CHECK();
    return GS_OK;
}
