// gs_sample.hip — indices drawn from given random numbers: rows of logits (or opacity logits), temperature, top-k,
// top-p, min-p.  C ABI: include/gsplat_densify.h (gs_sample), which also holds the definition.
//
//   order   entries by descending value, equal ones by ascending index; NaN and -inf are no candidates
//   weight  w = exp((l - max l) / T), l = x, or log sigmoid(x) for opacity logits
//   kept    the first k of the order; of these the shortest prefix whose mass reaches p times theirs; of these w >= min_p
//   draw    the lowest index whose running sum of kept weights, in index order, exceeds u times the total
//
// The kept entries are a prefix of the order up to min_p, so a row's selection is two numbers: a threshold key and how
// many of the entries that equal it are kept (the lowest indices).  Keys are the value's bits mapped so that unsigned
// order is value order (a 16-bit type's key sits in the upper half); 0 stands for "no candidate".  A threshold is found
// digit by digit (11, 11, 10 bits from the top): a histogram of counts (top-k) or of masses (top-p) over the digit among
// the entries that agree with the digits found, and the digit in which the running total from above reaches its goal.
// Nothing is sorted.
//
// Weights are 64-bit: an index is right or wrong, and with 5 million candidates and 250 000 draws a 24-bit weight would
// move a border across a draw several times in every call.  Their sums are integers: a weight is rounded once, so that
// sums have no order, running sums never decrease, and a histogram's total, a chunk's and a draw's agree to the last bit.
//   up to 8192 entries   one word: multiples of 2^-50 of the row's largest (2^-49 beyond 4096 entries)
//   longer               two words: multiples of 2^-(124 - 2 c), c = ceil log2 cols: 2^-80 at 4 M entries.  One word's 2^-40
//                        there is not enough: 4 M entries that weigh e^-15 beside a peak are off by 2^-19 each, all the same
//                        way, and one draw in eight of the tail's lands on another index
//
// Two forms, by the length of a row:
//   up to 8192 entries: one workgroup per row does everything, the entries in its registers (k_sample_row); with many draws
//   several, each with the whole selection
//   longer: the row is cut into chunks of 4096 over the whole chip, and a launch per step (k_long_*).  With top-k, rows
//   whose candidates behind the first digit number 8192 or fewer are listed, if they have few draws, and go on as a short
//   row does (k_long_list)
//
// Measured (kernels, MI355X): 28 entries 4.8 us; 28 rows of 8160 with top-p 14.4 us; 1 M opacities, 50 000 draws 22 us (max
// 2.9, sums 8.3 .. 9.4, scan 2.0 .. 3.9, draws 8.0); 5 M opacities at a temperature with top-p, 250 000 draws 128 us (digits
// 27 + 20 + 10, sums 24, draws 31, the rest 16); 64 rows of 131072 bfloat16 with top-k and top-p 60 us a call (first digit 9,
// lists 17, the listed rows 20, the launches for others 2 .. 5 each).  The second word of a weight is 10 to 20 % of a long
// row's time (calls: 1 M 18 -> 20 us, 5 M 111 -> 115 .. 120, 64 x 131072 float32 with top-p 70 -> 81).  A pass over 5 M entries
// at the memory's rate is 5 us: the digits and sums of powers are bound by fp64 issue (80 instructions an entry, 10 us a pass
// at the peak rate) and the fixed 6 to 9 us of a launch that picks a digit, reads a row from the caches and adds up a
// histogram.
#include <math.h>

#include <type_traits>

#include "gs_device.h"
#include "../../include/gsplat_densify.h"

namespace gs {

enum SampleDtype { kF32 = GS_DTYPE_F32, kF16 = GS_DTYPE_F16, kBF16 = GS_DTYPE_BF16 };

struct SampleArgs {
    const void *logits;
    int64_t stride;
    int rows, cols, draws;
    double unit;                               // one workgroup: a weight of 1 as an integer, 2^50 or 2^49
    double high;                               // longer rows: 2^bits, cols * high <= 2^62; a weight of 1 is high * high
    int bits;
    GsSampleConfig cfg;
};

// A row's settings.  `greedy`: the first of the order alone (largest value, lowest index).
struct RowSettings {
    double inv_t, top_p, min_p;
    int top_k;                                 // 0: all
    bool ok, greedy;
};

static __device__ __forceinline__ RowSettings row_settings(const SampleArgs &a, int r) {
    const GsSampleConfig &c = a.cfg;
    const float t = c.temperature_rows ? c.temperature_rows[r] : c.temperature;
    const float p = c.top_p_rows ? c.top_p_rows[r] : c.top_p;
    const float m = c.min_p_rows ? c.min_p_rows[r] : c.min_p;
    const int k = c.top_k_rows ? c.top_k_rows[r] : c.top_k;
    RowSettings s;
    s.ok = t >= 0.0f && !isnan(p) && !isnan(m);
    s.greedy = t == 0.0f || m > 1.0f || p <= 0.0f || k == 1;
    s.top_k = (k > 0 && k < a.cols) ? k : 0;
    s.inv_t = s.greedy ? 1.0 : 1.0 / (double)t;
    s.top_p = p < 1.0f ? (double)p : 1.0;
    s.min_p = s.greedy ? 0.0 : (double)m;
    return s;
}

// ---- keys -------------------------------------------------------------------------------------------------------
static __device__ __forceinline__ uint32_t key_f32(uint32_t b) {
    const float x = __uint_as_float(b);
    if (!(x > -INFINITY)) return 0u;           // NaN, -inf
    b = __float_as_uint(x + 0.0f);             // (-0 and 0 are equal values)
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// 16-bit types: `b` the raw bits, `inf` the bits of +inf (all beyond it are NaN)
template <int DT>
static __device__ __forceinline__ uint32_t key_16(uint32_t b) {
    constexpr uint32_t inf = DT == kBF16 ? 0x7F80u : 0x7C00u;
    if ((b & 0x7FFFu) > inf || b == (inf | 0x8000u)) return 0u;
    if (b == 0x8000u) b = 0u;
    return ((b & 0x8000u) ? (~b & 0xFFFFu) : (b | 0x8000u)) << 16;
}
template <int DT>
static __device__ __forceinline__ float value_of(uint32_t key) {
    if constexpr (DT == kF32) return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
    const uint32_t h = key >> 16, b = (h & 0x8000u) ? (h & 0x7FFFu) : (~h & 0xFFFFu);
    if constexpr (DT == kBF16) return __uint_as_float(b << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}
template <int DT>
constexpr int kBytes = DT == kF32 ? 4 : 2;
template <int DT>
constexpr int kVec = 16 / kBytes<DT>;          // entries of one 16-byte load (of any alignment)

template <int DT>
static __device__ __forceinline__ uint32_t key_at(const char *row, int64_t i) {
    if constexpr (DT == kF32) {
        return key_f32(reinterpret_cast<const uint32_t *>(row)[i]);
    } else {
        return key_16<DT>(reinterpret_cast<const uint16_t *>(row)[i]);
    }
}
// keys of entries i .. i + kVec - 1 (0 behind the row's end)
template <int DT>
static __device__ __forceinline__ void keys_at(const char *row, int64_t i, int64_t n, uint32_t (&k)[kVec<DT>]) {
    if (i + kVec<DT> <= n) {
        uint32_t w[4];
        __builtin_memcpy(w, row + i * kBytes<DT>, 16);
#pragma unroll
        for (int e = 0; e < kVec<DT>; e++) {
            if constexpr (DT == kF32) {
                k[e] = key_f32(w[e]);
            } else {
                k[e] = key_16<DT>((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < kVec<DT>; e++) k[e] = i + e < n ? key_at<DT>(row, i + e) : 0u;
    }
}

// ---- weights ----------------------------------------------------------------------------------------------------
// p * x + c with the constant in scalar registers: left to itself the compiler takes the two-address form and copies every
// coefficient of a polynomial into vector registers first, one instruction in six of a weight.
static __device__ __forceinline__ double fma_const(double p, double x, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(p), "v"(x), "s"(c));
    return r;
}

// 2^y for y <= 0: 2^n times the polynomial that agrees with 2^f at the eleven Chebyshev nodes of |f| <= 1/2 (3e-16
// relative).  Adding 1.5 2^52 rounds y to the integer n and leaves n in the low word; it goes into the exponent by an
// integer addition.  Below 2^-1000: 2^-1000.
static __device__ __forceinline__ double pow2(double y) {
    y = fmax(y, -1000.0);
    const double shifted = y + 0x1.8p52, f = y - (shifted - 0x1.8p52);
    const int n = (int)(uint32_t)__double_as_longlong(shifted);
    double p = 0x1.e6063f7217bc6p-28;
    p = fma_const(p, f, 0x1.b675bca4eeebbp-24);
    p = fma_const(p, f, 0x1.62bfd47773353p-20);
    p = fma_const(p, f, 0x1.ffcb54062e698p-17);
    p = fma_const(p, f, 0x1.430913096fd9fp-13);
    p = fma_const(p, f, 0x1.5d87fe9d7a584p-10);
    p = fma_const(p, f, 0x1.3b2ab6fba1ddap-7);
    p = fma_const(p, f, 0x1.c6b08d703ce49p-5);
    p = fma_const(p, f, 0x1.ebfbdff82c598p-3);
    p = fma_const(p, f, 0x1.62e42fefa3a19p-1);
    p = fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + (n << 20), __double2loint(p));
}
constexpr double kLog2e = 1.4426950408889634073599246810019;

static __device__ __forceinline__ double reciprocal(double d) {   // d in [1, 2] (or a few times that)
    double r = __builtin_amdgcn_rcp(d);
    r = fma(fma(-d, r, 1.0), r, r);
    return fma(fma(-d, r, 1.0), r, r);
}
// log(1 + z), z in [0, 1]: 2 atanh(s) = 2 s (1 + q h(q)) with s = z / (2 + z) <= 1/3, q = s^2, and h by its polynomial
// through ten Chebyshev nodes of [0, 1/9] (2e-16 relative, of which q h passes on a twenty-fifth)
static __device__ __forceinline__ double log1p_unit(double z) {
    const double s = z * reciprocal(2.0 + z), q = s * s;
    double p = 0x1.4b0a26c5f2aefp-4;
    p = fma_const(p, q, 0x1.687a6e7c95176p-5);
    p = fma_const(p, q, 0x1.eb905e8575054p-5);
    p = fma_const(p, q, 0x1.10ac75dc602b1p-4);
    p = fma_const(p, q, 0x1.3b18b294bebf9p-4);
    p = fma_const(p, q, 0x1.745cf0b0e03bdp-4);
    p = fma_const(p, q, 0x1.c71c727143318p-4);
    p = fma_const(p, q, 0x1.24924923d44c6p-3);
    p = fma_const(p, q, 0x1.999999999a3ddp-3);
    p = fma_const(p, q, 0x1.5555555555555p-2);
    return 2.0 * fma(p * q, s, s);
}
template <bool OPACITY>
static __device__ __forceinline__ double log_weight(double x) {
    if constexpr (!OPACITY) return x;
    return fmin(x, 0.0) - log1p_unit(pow2(-fabs(x) * kLog2e));
}

// Weights relative to the key `top` (its own is 1).
struct Scale {
    double l_top, rate, norm;                  // rate = log2(e) / T;  norm = 1 / sigmoid(top)
    uint32_t top;
    bool unit;                                 // opacities at temperature 1: w = sigmoid(x) * norm
};
template <int DT, bool OPACITY>
static __device__ __forceinline__ Scale scale_for(uint32_t top, double inv_t) {
    Scale s;
    const double x = (double)value_of<DT>(top);
    s.top = top;
    s.l_top = log_weight<OPACITY>(x);
    s.rate = inv_t * kLog2e;
    // (further down, pow2's least value times this norm would be a weight: 2^-1000 e^300 is none, 2^-1000 e^690 is 0.04)
    s.unit = OPACITY && inv_t == 1.0 && x > -300.0;
    s.norm = s.unit ? 1.0 + exp(-x) : 1.0;
    return s;
}
template <int DT, bool OPACITY>
static __device__ __forceinline__ double weight(uint32_t key, const Scale &s) {
    if (key == s.top) return 1.0;              // (also +inf - +inf)
    const double x = (double)value_of<DT>(key);
    if constexpr (OPACITY) {
        if (s.unit) {
            const double z = pow2(-fabs(x) * kLog2e);
            return fmin((x < 0.0 ? z : 1.0) * reciprocal(1.0 + z) * s.norm, 1.0);
        }
    }
    return pow2((log_weight<OPACITY>(x) - s.l_top) * s.rate);
}
// ---- digits of a threshold ----------------------------------------------------------------------------------------
constexpr int kBins = 2048;
constexpr int kLevels = 3;
template <int DT>
constexpr int kUsedLevels = DT == kF32 ? 3 : 2;   // a 16-bit type's key ends within the second digit
static __device__ __forceinline__ int digit_shift(int level) { return level == 0 ? 21 : (level == 1 ? 10 : 0); }
static __device__ __forceinline__ uint32_t digit_of(uint32_t key, int level) {
    return level == 0 ? key >> 21 : (level == 1 ? (key >> 10) & 2047u : key & 1023u);
}
// the digits above `level` of `key` are those found
static __device__ __forceinline__ bool agrees(uint32_t key, uint32_t found, int level) {
    return level == 0 || (key >> (level == 1 ? 21 : 10)) == (found >> (level == 1 ? 21 : 10));
}

// A search, for top-k (counts) or top-p (masses), as it stands between two digits.
template <typename SUM, typename GOAL>
struct SearchOf {
    SUM above;                                 // count or mass over the digits found
    GOAL goal;                                 // count or mass to reach
    uint32_t found;
    uint32_t done;                             // nothing to cut: every candidate is kept
};
using Search = SearchOf<uint64_t, double>;

// Masses of the longer rows, in units of 1 / high^2.
using Mass = uint128;
using MassSearch = SearchOf<Mass, Mass>;

// A weight as high * hi + lo, |lo| <= high / 2: sums of either word over a row stay below 2^63, without carries.
struct Words {
    uint64_t hi;
    int64_t lo;
};
static __device__ __forceinline__ Words words_of(double w, double high) {
    const double h = fma(w, high, 0x1p52), l = fma(fma(w, high, -(h - 0x1p52)), high, 0x1.8p52);
    return {(uint64_t)__double_as_longlong(h) - 0x4330000000000000ull,
            (int64_t)((uint64_t)__double_as_longlong(l) - 0x4338000000000000ull)};
}
static __device__ __forceinline__ Mass mass_of(const Words &v, int bits) { return ((Mass)v.hi << bits) + (Mass)(__int128)v.lo; }
static __device__ __forceinline__ double as_double(Mass v) { return (double)(uint64_t)(v >> 64) * 0x1p64 + (double)(uint64_t)v; }

// floor (or ceiling) of f * total without a rounding; 0 <= f < 1, total < 2^112
static __device__ __forceinline__ Mass share_of(Mass total, float f, bool up) {
    const uint32_t b = __float_as_uint(f) & 0x7FFFFFFFu, e = b >> 23;   // (-0 is 0)
    const uint64_t m = e ? (b & 0x7FFFFFu) | 0x800000u : b & 0x7FFFFFu;
    const int k = e ? 150 - (int)e : 149;      // f = m 2^-k, 24 <= k
    const Mass low = (Mass)(uint64_t)total * m, x = (Mass)(uint64_t)(total >> 64) * m + (uint64_t)(low >> 64);
    const uint64_t y = (uint64_t)low;          // f * total = (x 2^64 + y) 2^-k, x < 2^73
    Mass q;
    bool rest;
    if (k < 64) {
        q = (x << (64 - k)) | (y >> k);
        rest = (y << (64 - k)) != 0;
    } else {
        q = x >> (k - 64);
        rest = y != 0 || x != (q << (k - 64));
    }
    return q + (up && rest ? 1u : 0u);
}

// w * unit <= 2^50, rounded to the nearest integer: the low bits of that number plus 2^52
static __device__ __forceinline__ uint64_t fixed(double w, double unit) {
    return (uint64_t)__double_as_longlong(fma(w, unit, 0x1p52)) - 0x4330000000000000ull;
}

// A lane's value as one that the wave has in common, in scalar registers: `lane` is in common too.
static __device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
static __device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
    return (uint64_t)lane_value((uint32_t)v, lane) | (uint64_t)lane_value((uint32_t)(v >> 32), lane) << 32;
}
static __device__ __forceinline__ Mass lane_value(Mass v, int lane) {
    return (Mass)lane_value((uint64_t)v, lane) | (Mass)lane_value((uint64_t)(v >> 64), lane) << 64;
}
static __device__ __forceinline__ Mass shuffle(Mass v, int lane) {
    return (Mass)__shfl((uint64_t)v, lane, 64) | (Mass)__shfl((uint64_t)(v >> 64), lane, 64) << 64;
}

// Exclusive scan over the workgroup in thread order, THREADS a multiple of 64 up to 1024; `total` gets the sum.  Each wave
// scans the waves' sums in its first lanes: added up one after the other they were 16 times eight instructions of every wave
// where a sum has four words.
template <int THREADS, typename T>
static __device__ __forceinline__ T block_scan(T v, T *wave_sums /* LDS [THREADS / 64] */, T &total) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const T s = wave_scan(v), before = s - v;
    if constexpr (THREADS == 64) {
        total = lane_value(s, 63);
        return before;
    }
    static_assert(THREADS <= 1024, "a row of lanes");
    __syncthreads();
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    const T one = lane < THREADS / 64 ? wave_sums[lane] : T(0), upto = row_scan(one);
    total = lane_value(upto, THREADS / 64 - 1);
    return before + lane_value(upto - one, wave);
}

static __device__ __forceinline__ bool below(uint64_t sum, double goal) { return (double)sum < goal; }
static __device__ __forceinline__ bool below(Mass sum, Mass goal) { return sum < goal; }

// The digit in which the running total, from the largest digit down, reaches the goal (kBins: none does).  `bin(i)`: count
// or mass of digit i; `goal_of_total(t)`: the goal, where all the digits together hold t.  Every thread of the workgroup gets
// the digit and what lies above it (all, if none does); called with the histogram complete, each time with a place `out` of
// its own.
template <typename SUM>
struct PickedOf {
    uint32_t digit;
    SUM above, total;
};
using Picked = PickedOf<uint64_t>;
template <int THREADS, typename SUM, typename F, typename G>
static __device__ PickedOf<SUM> pick_digit(F bin, SUM above, G goal_of_total, SUM *wave_sums, PickedOf<SUM> *out /* LDS */) {
    constexpr int per = kBins / THREADS < 1 ? 1 : kBins / THREADS;
    const int tid = threadIdx.x, high = kBins - 1 - tid * per;
    if (tid == 0) out->digit = kBins;          // (the scan's barriers stand between this and the writer below)
    SUM mine = 0;
#pragma unroll 4
    for (int j = 0; j < per; j++) mine += bin(high - j);
    SUM total;
    SUM run = above + block_scan<THREADS>(mine, wave_sums, total);
    const auto need = goal_of_total(total);
    // the one thread whose part crosses: its start is below the goal, its end is not
    if (below(run, need) && !below(run + mine, need) && mine > 0) {
        for (int j = 0; j < per; j++) {
            const SUM b = bin(high - j);
            if (b > 0 && !below(run + b, need)) {
                out->digit = (uint32_t)(high - j);
                out->above = run;
                break;
            }
            run += b;
        }
    }
    __syncthreads();
    if (out->digit == kBins) return {kBins, above + total, total};
    return {out->digit, out->above, total};
}

static __device__ __forceinline__ uint32_t ties_for(uint64_t above, double goal, double tie_weight, double unit,
                                                    uint64_t have) {  // (one word)
    const double w = (double)fixed(tie_weight, unit);
    const double n = w > 0.0 ? ceil((goal - (double)above) / w) : (double)have;
    return (uint32_t)fmin(fmax(n, 1.0), (double)have);
}

// The least number of ties that reaches the goal, 1 .. have; `tie`: the mass of one
static __device__ __forceinline__ uint32_t ties_for(Mass above, Mass goal, Mass tie, uint64_t have) {
    const Mass lack = goal - above;
    uint64_t n = (uint64_t)fmin(tie > 0 ? as_double(lack) / as_double(tie) : (double)have, (double)have);
    if (n < 1) n = 1;
    while (n < have && tie * n < lack) n++;    // (the quotient is good to a few 2^-52: a step or two)
    while (n > 1 && tie * (n - 1) >= lack) n--;
    return (uint32_t)n;
}

// floor(u * total), below total: the running sums that exceed u * total are those that exceed it
static __device__ __forceinline__ uint64_t goal_of(float u, uint64_t total) {
    const double g = fmax((double)u, 0.0) * (double)total;
    return g < (double)total ? min((uint64_t)g, total - 1) : total - 1;
}
static __device__ __forceinline__ Mass goal_of(float u, Mass total) {
    return u < 1.0f ? share_of(total, fmaxf(u, 0.0f), false) : total - 1;
}

// ---- rows of up to 8192 entries ------------------------------------------------------------------------------------
constexpr int kEach = 8;                       // entries per thread

// A workgroup's memory for the selection among up to 8 THREADS entries.  Histograms: 1024 threads have one for every
// digit, emptied together, which saves two barriers of sixteen waves a digit, and the first digit's masses in copies by lane
// (neighbouring values share it, a wave's atomics would hit few words).  Fewer threads: one for all, so that many short
// rows share a compute unit.  The first words also hold, in turn, the weights of entry 8 t + e at [e][t], 0 if it is not
// kept; the counts' the running sums.
template <int THREADS>
struct RowShared {
    static constexpr bool kSplit = THREADS >= 1024;
    static constexpr int kPitch = THREADS + 1, kCopies = THREADS >= 1024 ? 4 : 1;
    static constexpr int kFirst = kEach * kPitch > kBins * kCopies ? kEach * kPitch : kBins * kCopies;
    uint64_t masses[kFirst + (kSplit ? (kLevels - 1) * kBins : 0)];
    uint64_t counts_or_sums[(kSplit ? kLevels + 1 : 1) * kBins / 2];
    uint64_t waves_u[THREADS / 64];
    uint32_t waves_i[THREADS / 64];
    Picked picks[2 * kLevels];
};

// A row's selection and its draws, by one workgroup; thread t holds the keys of entries 8 t .. 8 t + 7, so that thread order
// is index order.  `mx`: the largest key, not 0.  `f_k`: the search of top-k as it stands before digit `level_k`.  Of the
// draws, those of `part` of `parts`.  `index(i)`: the index in the row of entry i.
template <int DT, bool OPACITY, int THREADS, typename F>
static __device__ __forceinline__ void draw_row(const SampleArgs &a, const RowSettings &set, int r, const uint32_t (&key)[kEach],
                                                uint32_t mx, Search f_k, int level_k, int part, int parts,
                                                RowShared<THREADS> &sh, const float *__restrict__ uniforms,
                                                int32_t *__restrict__ ids, F index) {
    constexpr bool kSplit = RowShared<THREADS>::kSplit;
    constexpr int kPitch = RowShared<THREADS>::kPitch, kRowCopies = RowShared<THREADS>::kCopies;
    constexpr int kFirst = RowShared<THREADS>::kFirst;
    uint64_t *masses = sh.masses, *kept_w = sh.masses, *run_sum = sh.counts_or_sums, *waves_u = sh.waves_u;
    uint32_t *counts = reinterpret_cast<uint32_t *>(sh.counts_or_sums), *waves_i = sh.waves_i;
    Picked *picks = sh.picks;
    const int tid = threadIdx.x;
    const Scale s = scale_for<DT, OPACITY>(mx, set.inv_t);
    double w[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        w[e] = 0.0;
        if (key[e] != 0 && (!set.greedy || key[e] == mx)) w[e] = weight<DT, OPACITY>(key[e], s);
    }
    uint32_t thr = 0, ties = 0;
    const bool with_k = !set.greedy && set.top_k > 0, with_p = !set.greedy && set.top_p < 1.0;
    if (kSplit && (with_k || with_p)) {
        if (with_p)
            for (int b = tid; b < kBins * kRowCopies; b += THREADS) masses[b] = 0;
        if (with_p)
            for (int b = tid; b < (kLevels - 1) * kBins; b += THREADS) masses[kFirst + b] = 0;
        for (int b = tid; b < (kLevels + 1) * kBins; b += THREADS) counts[b] = 0;
        __syncthreads();
    }
    if (with_k) {
        Search f = f_k;
        for (int level = level_k; level < kUsedLevels<DT> && !f.done; level++) {
            uint32_t *count = counts + (kSplit ? level * kBins : 0);
            if (!kSplit) {
                __syncthreads();
                for (int b = tid; b < kBins; b += THREADS) count[b] = 0;
                __syncthreads();
            }
#pragma unroll
            for (int e = 0; e < kEach; e++)
                if (key[e] != 0 && agrees(key[e], f.found, level)) atomicAdd(&count[digit_of(key[e], level)], 1u);
            __syncthreads();
            const Picked p = pick_digit<THREADS>([&](int i) { return (uint64_t)count[i]; }, f.above,
                                                 [&](uint64_t) { return f.goal; }, waves_u, &picks[level]);
            if (p.digit == kBins) f.done = 1;  // fewer candidates than k
            else f.found |= p.digit << digit_shift(level);
            f.above = p.above;
        }
        if (!f.done) {
            thr = f.found;
            ties = (uint32_t)set.top_k - (uint32_t)f.above;
        }
    }
    if (with_p) {
        const uint32_t kthr = thr, kties = ties;
        uint64_t tied = 0;                     // the ties that top-k left, as one
        if (kthr) tied = (uint64_t)kties * fixed(weight<DT, OPACITY>(kthr, s), a.unit);
        Search f = {0, 0.0, 0, 0};
        uint64_t have = 0;
        for (int level = 0; level < kUsedLevels<DT>; level++) {
            uint64_t *mass = masses + (kSplit && level > 0 ? kFirst + (level - 1) * kBins : 0);
            uint32_t *count = counts + (kSplit ? kLevels * kBins : 0);
            const int copies = level == 0 ? kRowCopies : 1;
            if (!kSplit) {
                __syncthreads();
                for (int b = tid; b < kBins; b += THREADS) {
                    mass[b] = 0;
                    count[b] = 0;
                }
                __syncthreads();
            }
            uint64_t *copy = mass + (tid & (copies - 1)) * kBins;
            const bool last = level == kUsedLevels<DT> - 1;
            auto add = [&](uint32_t k, uint64_t w_, uint32_t n_) {
                const uint32_t d = digit_of(k, level);
                atomicAdd((unsigned long long *)&copy[d], (unsigned long long)w_);
                if (last) atomicAdd(&count[d], n_);
            };
#pragma unroll
            for (int e = 0; e < kEach; e++)
                if (key[e] > kthr && agrees(key[e], f.found, level)) add(key[e], fixed(w[e], a.unit), 1u);
            if (tid == 0 && kthr && agrees(kthr, f.found, level)) add(kthr, tied, kties);
            __syncthreads();
            const Picked p = pick_digit<THREADS>([&](int i) {
                uint64_t m = mass[i];
                for (int c = 1; c < copies; c++) m += mass[c * kBins + i];
                return m;
            }, f.above, [&](uint64_t t) { return level == 0 ? set.top_p * (double)t : f.goal; }, waves_u,
                                                 &picks[kLevels + level]);
            if (level == 0) f.goal = set.top_p * (double)p.total;
            if (p.digit == kBins) {            // (nothing weighs anything in fixed point but the first)
                f.done = 1;
                break;
            }
            f.found |= p.digit << digit_shift(level);
            f.above = p.above;
            if (last) have = count[p.digit];
        }
        if (!f.done) {
            thr = f.found;
            ties = ties_for(f.above, f.goal, weight<DT, OPACITY>(thr, s), a.unit, have);
        }
    }
    __syncthreads();
    // what is kept: ties by their rank in index order
    uint32_t rank = 0;
    if (thr) {
        uint32_t mine = 0, all;
#pragma unroll
        for (int e = 0; e < kEach; e++) mine += key[e] == thr;
        rank = block_scan<THREADS>(mine, waves_i, all);
    }
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const bool tied = thr != 0 && key[e] == thr;
        const bool keep = key[e] > thr || (tied && rank < ties);
        rank += tied;
        const uint64_t v = (keep && w[e] >= set.min_p) ? fixed(w[e], a.unit) : 0ull;
        kept_w[e * kPitch + tid] = v;
        sum += v;
    }
    uint64_t total;
    run_sum[tid] = block_scan<THREADS>(sum, waves_u, total);
    __syncthreads();
    for (int64_t j = (int64_t)part * THREADS + tid; j < a.draws; j += (int64_t)parts * THREADS) {
        const float u = uniforms[(size_t)r * a.draws + j];
        const uint64_t goal = set.greedy ? 0ull : goal_of(u, total);
        int lo = 0, hi = THREADS;              // run_sum[lo] <= goal < run_sum[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (run_sum[mid] <= goal) lo = mid;
            else hi = mid;
        }
        uint64_t c = run_sum[lo];
        int e = -1;
        do c += kept_w[++e * kPitch + lo];
        while (c <= goal && e < kEach - 1);
        ids[(size_t)r * a.draws + j] = isnan(u) ? -1 : index(lo * kEach + e);
    }
}

// `parts` workgroups per row, each with a share of its draws; the selection is each one's own.  Bound by latency: a dozen
// barriers, and per digit one LDS atomic an entry; the entries are read once.
template <int DT, bool OPACITY, int THREADS>
__global__ void __launch_bounds__(THREADS)
k_sample_row(SampleArgs a, int parts, const float *__restrict__ uniforms, int32_t *__restrict__ ids) {
    __shared__ RowShared<THREADS> sh;
    const int r = blockIdx.x / parts, part = blockIdx.x - r * parts, tid = threadIdx.x, n = a.cols;
    const char *row = static_cast<const char *>(a.logits) + (size_t)r * a.stride * kBytes<DT>;
    const RowSettings set = row_settings(a, r);
    uint32_t key[kEach];
#pragma unroll
    for (int q = 0; q < kEach / kVec<DT>; q++) {
        uint32_t k[kVec<DT>];
        keys_at<DT>(row, (int64_t)tid * kEach + q * kVec<DT>, n, k);
#pragma unroll
        for (int e = 0; e < kVec<DT>; e++) key[q * kVec<DT> + e] = k[e];
    }
    uint32_t mx = 0;
#pragma unroll
    for (int e = 0; e < kEach; e++) mx = max(mx, key[e]);
    for (int off = 32; off > 0; off >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, off, 64));
    if constexpr (THREADS > 64) {
        if ((tid & 63) == 0) sh.waves_i[tid >> 6] = mx;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; w++) mx = max(mx, sh.waves_i[w]);
    }
    if (!set.ok || mx == 0) {
        for (int64_t j = (int64_t)part * THREADS + tid; j < a.draws; j += (int64_t)parts * THREADS)
            ids[(size_t)r * a.draws + j] = -1;
        return;
    }
    draw_row<DT, OPACITY, THREADS>(a, set, r, key, mx, {0, (double)set.top_k, 0, 0}, 0, part, parts, sh, uniforms, ids,
                                   [](int i) { return i; });
}

// ---- longer rows ------------------------------------------------------------------------------------------------------
constexpr int kSeg = 8;                        // entries between two stored running sums
constexpr int kChunkThreads = 512;             // (8 entries a thread: a million entries are two waves a SIMD)
constexpr int kChunk = kChunkThreads * kSeg;
constexpr int kChunkSegs = kChunkThreads;
constexpr int kHistThreads = 1024;
constexpr int kBatch = 2;                      // loads a thread of a digit's launch has in flight
constexpr int kCopies = 2;
constexpr int kQueue = 576;                    // keys a wave can have waiting
constexpr int kListThreads = 1024;
constexpr int kListMax = kListThreads * kEach; // entries of a row that one workgroup takes over
constexpr int kListPitch = 32;
constexpr int kRun = 256;                      // entries of a row that the shortest run in a list spans
constexpr int kRunMax = 8192;                  // runs of a row
template <int DT>
constexpr int kWaveEntries = 64 * kVec<DT>;    // entries of a wave's load: a run

// A row's state between the launches.  A launch reads what earlier ones wrote and writes other fields.
struct LongRow {
    double inv_t, top_p, min_p;
    Scale scale;
    Mass total, tie_weight;
    MassSearch p[kLevels];                     // as the launch of that digit found it (a listed row's k[0]: as it left it)
    Search k[kLevels];
    uint32_t k_thr, k_ties, thr, ties;
    int32_t top_k;
    uint32_t ok, greedy;
    uint32_t listed;                           // entries in the row's list; 0: the row has none
};

struct LongArgs {
    LongRow *rows;
    uint32_t *k_count;                         // [rows][kLevels][kBins]
    uint64_t *p_mass;                          // [rows][kLevels][2][kBins]: the high words' sums, the low words'
    uint32_t *p_count;                         // [rows][kBins], of the last digit
    uint32_t *chunk_max;                       // [rows][chunks], of which `maxima` are used
    Mass *chunk_sum;                           // [rows][chunks]: sums, then running sums
    uint32_t *chunk_ties;                      // [rows][chunks]: ties, then running ties
    Mass *seg_sum;                             // [rows][chunks][kChunkSegs] running sums inside the chunk
    Mass *mid_sum, *top_sum;                   // every 8th and every 64th of them again, for the draws' first steps
    uint32_t *seg_ties;                        // [rows][chunks][kChunkSegs]
    uint2 *list;                               // [rows][kListMax]: key, index
    int32_t *list_index;                       // [rows][kListMax]: in order
    uint32_t *list_runs;                       // [rows][run_pitch]: a run's place in the list | its entries << 16
    uint32_t *list_count;                      // [rows][kListPitch], the first of each: a line of its own
    int chunks, maxima, run_pitch;
    bool with_k, with_p;                       // launches that look for a threshold
    bool lists;                                // a row's candidates for top-k may be listed
};

template <int DT>
static __device__ __forceinline__ const char *row_base(const SampleArgs &a, int r) {
    return static_cast<const char *>(a.logits) + (size_t)r * a.stride * kBytes<DT>;
}

template <int DT>
static __device__ __forceinline__ void empty_p(const LongArgs &g, int r, int from, int step) {
    for (int b = from; b < kUsedLevels<DT> * 2 * kBins; b += step) {
        g.p_mass[(size_t)r * kLevels * 2 * kBins + b] = 0;
        if (b < kBins) g.p_count[(size_t)r * kBins + b] = 0;
    }
}

// A chunk's maximum; the histograms of top-p are emptied on the way.
template <int DT>
__global__ void __launch_bounds__(kChunkThreads)
k_long_max(SampleArgs a, LongArgs g) {
    __shared__ uint32_t waves[kChunkThreads / 64];
    const int r = blockIdx.x / g.chunks, c = blockIdx.x - r * g.chunks, tid = threadIdx.x;
    const char *row = row_base<DT>(a, r);
    uint32_t mx = 0;
#pragma unroll
    for (int q = 0; q < kSeg / kVec<DT>; q++) {
        uint32_t k[kVec<DT>];
        keys_at<DT>(row, (int64_t)c * kChunk + ((int64_t)q * kChunkThreads + tid) * kVec<DT>, a.cols, k);
#pragma unroll
        for (int e = 0; e < kVec<DT>; e++) mx = max(mx, k[e]);
    }
    if (g.with_p) empty_p<DT>(g, r, c * kChunkThreads + tid, g.chunks * kChunkThreads);
    for (int off = 32; off > 0; off >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, off, 64));
    if ((tid & 63) == 0) waves[tid >> 6] = mx;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < kChunkThreads / 64; w++) mx = max(mx, waves[w]);
        g.chunk_max[(size_t)r * g.chunks + c] = mx;
    }
}

// The row's settings and maximum, nothing cut yet.
template <int DT, bool OPACITY>
static __device__ __forceinline__ LongRow long_row(const SampleArgs &a, int r, uint32_t max_key) {
    const RowSettings set = row_settings(a, r);
    LongRow s = {};
    s.inv_t = set.inv_t;
    s.top_p = set.top_p;
    s.min_p = set.min_p;
    s.top_k = set.top_k;
    s.ok = set.ok && max_key != 0;
    s.greedy = set.greedy;
    s.scale = scale_for<DT, OPACITY>(max_key, set.inv_t);
    s.k[0].goal = set.greedy ? 1.0 : (double)set.top_k;
    s.k[0].done = !s.ok || (!set.greedy && set.top_k == 0);
    s.p[0].done = set.greedy || !s.ok || !(set.top_p < 1.0);
    return s;
}

// Maximum over the row's parts, by every workgroup for itself.
template <int THREADS>
static __device__ __forceinline__ uint32_t row_max(const LongArgs &g, int r, uint32_t *waves /* LDS [THREADS / 64] */) {
    uint32_t mx = 0;
    for (int c = threadIdx.x; c < g.maxima; c += THREADS) mx = max(mx, g.chunk_max[(size_t)r * g.chunks + c]);
    for (int off = 32; off > 0; off >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, off, 64));
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) mx = max(mx, waves[w]);
    __syncthreads();
    return mx;
}

// With top-k: empty histograms and lists.
template <int DT>
__global__ void __launch_bounds__(kHistThreads)
k_long_empty(LongArgs g, int parts) {
    const int r = blockIdx.x / parts, part = blockIdx.x - r * parts;
    const int from = part * kHistThreads + threadIdx.x, step = parts * kHistThreads;
    for (int b = from; b < kUsedLevels<DT> * kBins; b += step) g.k_count[(size_t)r * kLevels * kBins + b] = 0;
    if (g.with_p) empty_p<DT>(g, r, from, step);
    if (g.lists) {
        for (int b = from; b < g.run_pitch; b += step) g.list_runs[(size_t)r * g.run_pitch + b] = 0;
        if (from == 0) g.list_count[(size_t)r * kListPitch] = 0;
    }
}

// With top-k: a part's maximum and the histogram of the first digit, which needs nothing else.
template <int DT>
__global__ void __launch_bounds__(kHistThreads)
k_long_first(SampleArgs a, LongArgs g, int parts) {
    __shared__ uint32_t count[kBins];
    __shared__ uint32_t waves[kHistThreads / 64];
    const int r = blockIdx.x / parts, part = blockIdx.x - r * parts, tid = threadIdx.x;
    const char *row = row_base<DT>(a, r);
    const int64_t n = a.cols, step = (int64_t)kHistThreads * kVec<DT>;
    for (int b = tid; b < kBins; b += kHistThreads) count[b] = 0;
    __syncthreads();
    uint32_t mx = 0;
    for (int64_t i0 = (int64_t)part * kBatch * step; i0 < n; i0 += (int64_t)parts * kBatch * step) {
        uint32_t k[kBatch][kVec<DT>];
#pragma unroll
        for (int q = 0; q < kBatch; q++) keys_at<DT>(row, i0 + (int64_t)tid * kVec<DT> + q * step, n, k[q]);
#pragma unroll
        for (int q = 0; q < kBatch; q++)
#pragma unroll
            for (int e = 0; e < kVec<DT>; e++) {
                mx = max(mx, k[q][e]);
                if (k[q][e]) atomicAdd(&count[digit_of(k[q][e], 0)], 1u);
            }
    }
    for (int off = 32; off > 0; off >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, off, 64));
    if ((tid & 63) == 0) waves[tid >> 6] = mx;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < kHistThreads / 64; w++) mx = max(mx, waves[w]);
        g.chunk_max[(size_t)r * g.chunks + part] = mx;
    }
    for (int b = tid; b < kBins; b += kHistThreads)
        if (count[b]) atomicAdd(&g.k_count[(size_t)r * kLevels * kBins + b], count[b]);
}

// Without top-k, one workgroup per row: its state.
template <int DT, bool OPACITY>
__global__ void __launch_bounds__(kHistThreads)
k_long_begin(SampleArgs a, LongArgs g) {
    __shared__ uint32_t waves[kHistThreads / 64];
    const uint32_t mx = row_max<kHistThreads>(g, blockIdx.x, waves);
    if (threadIdx.x == 0) g.rows[blockIdx.x] = long_row<DT, OPACITY>(a, blockIdx.x, mx);
}

// The state behind digit `level`, from its histogram; by every workgroup for itself, so that no launch waits for a last
// one.  `count` gets how many entries have that digit (top-p, last digit).
template <int DT>
static __device__ __forceinline__ Search after_k(const LongArgs &g, int r, int level, const Search &f, uint64_t *waves_u,
                                                 Picked *pick) {
    if (f.done) return f;
    const uint32_t *bins = g.k_count + ((size_t)r * kLevels + level) * kBins;
    const Picked p = pick_digit<kHistThreads>([&](int i) { return (uint64_t)bins[i]; }, f.above,
                                              [&](uint64_t) { return f.goal; }, waves_u, pick);
    Search next = f;
    if (p.digit == kBins) next.done = 1;       // fewer candidates than k
    else next.found |= p.digit << digit_shift(level);
    next.above = p.above;
    return next;
}
template <int DT, bool OPACITY>
static __device__ __forceinline__ MassSearch after_p(const SampleArgs &a, const LongArgs &g, int r, int level,
                                                     const MassSearch &f, const LongRow &st, uint32_t k_thr, uint32_t k_ties,
                                                     Mass *waves_m, PickedOf<Mass> *pick, uint64_t *have) {
    if (f.done) return f;
    // the ties that top-k left count as one entry of k_ties times the weight
    Mass tied = 0;
    int tied_digit = -1;
    if (k_thr && agrees(k_thr, f.found, level)) {
        tied = k_ties * mass_of(words_of(weight<DT, OPACITY>(k_thr, st.scale), a.high), a.bits);
        tied_digit = (int)digit_of(k_thr, level);
    }
    const uint64_t *bins = g.p_mass + ((size_t)r * kLevels + level) * 2 * kBins;
    const float share = (float)st.top_p;       // (as it was given)
    const PickedOf<Mass> p = pick_digit<kHistThreads>([&](int i) {
        return mass_of({bins[i], (int64_t)bins[kBins + i]}, a.bits) + (i == tied_digit ? tied : (Mass)0);
    }, f.above, [&](Mass t) { return level == 0 ? share_of(t, share, true) : f.goal; }, waves_m, pick);
    MassSearch next = f;
    if (level == 0) next.goal = share_of(p.total, share, true);
    if (p.digit == kBins) {
        next.done = 1;
    } else {
        next.found |= p.digit << digit_shift(level);
        next.above = p.above;
        *have = (uint64_t)g.p_count[(size_t)r * kBins + p.digit] + ((int)p.digit == tied_digit ? k_ties : 0u);
    }
    return next;
}
// The top-k threshold, once all its digits are counted.
template <int DT>
static __device__ __forceinline__ void finish_k(const LongArgs &g, int r, const LongRow &st, uint64_t *waves_u,
                                                Picked *pick, uint32_t &thr, uint32_t &ties) {
    constexpr int last = kUsedLevels<DT> - 1;
    thr = ties = 0;
    if (!g.with_k) return;
    const Search f = after_k<DT>(g, r, last, st.k[last], waves_u, pick);
    if (f.done) return;
    thr = f.found;
    ties = (uint32_t)f.goal - (uint32_t)f.above;
}

// The histogram of a digit of the top-k threshold (MASS false) or of the top-p threshold; `parts` workgroups per row.
// `first_launch`: none has prepared the rows' state, it is made here.  Where the candidates that the first digit leaves fit
// one workgroup, its second launch lists them instead, and k_long_list goes on with them: the row is read twice, not six
// or eight times.
// Bound by the loads' latency and by fp64: some 40 instructions a weight, 75 for an opacity's power.
template <int DT, bool OPACITY, bool MASS>
__global__ void __launch_bounds__(kHistThreads)
k_long_digit(SampleArgs a, LongArgs g, int parts, int level, bool first_launch) {
    // Neighbouring values share a first digit, a wave's atomics then hit few words: copies of the masses, by lane.
    constexpr int kMassWords = 2 * kBins * kCopies, kQueuedWords = 2 * kBins + kQueue * (kHistThreads / 64) / 2;
    __shared__ uint64_t mass[MASS ? (kMassWords > kQueuedWords ? kMassWords : kQueuedWords) : 1];
    __shared__ uint32_t count[kBins];
    __shared__ uint64_t waves_u[kHistThreads / 64];
    __shared__ Mass waves_m[MASS ? kHistThreads / 64 : 1];
    __shared__ PickedOf<Mass> pick_m;
    __shared__ uint32_t waves_i[kHistThreads / 64 * kBatch];
    __shared__ uint32_t list_at;
    __shared__ Picked pick;
    const int r = blockIdx.x / parts, part = blockIdx.x - r * parts, tid = threadIdx.x;
    LongRow &st = g.rows[r];
    if (!first_launch && (MASS ? st.p[0].done : st.k[1].done)) {
        if (MASS || level == 1 || part != 0 || tid != 0) return;
        st.k[level] = st.k[1];
        return;
    }
    // the first entries are under way while the digit before this one is picked
    const char *row = row_base<DT>(a, r);
    const int64_t n = a.cols, step = (int64_t)kHistThreads * kVec<DT>, first = (int64_t)part * kBatch * step;
    uint32_t k[kBatch][kVec<DT>];
#pragma unroll
    for (int q = 0; q < kBatch; q++) keys_at<DT>(row, first + (int64_t)tid * kVec<DT> + q * step, n, k[q]);
    uint32_t k_thr = 0, k_ties = 0;
    std::conditional_t<MASS, MassSearch, Search> f;
    Scale s;
    bool listed = false;
    if (first_launch) {
        const LongRow own = long_row<DT, OPACITY>(a, r, row_max<kHistThreads>(g, r, waves_i));
        if (part == 0 && tid == 0) st = own;
        s = own.scale;
        if constexpr (MASS) f = own.p[0];
        else f = own.k[0];
        if constexpr (!MASS) if (!f.done) {    // (level 1)
            f = after_k<DT>(g, r, 0, f, waves_u, &pick);
            const uint64_t n = f.above + (f.done ? 0 : g.k_count[(size_t)r * kLevels * kBins + digit_of(f.found, 0)]);
            listed = g.lists && n <= kListMax;
            if (listed && part == 0 && tid == 0) {
                st.listed = (uint32_t)n;
                st.k[0] = f;
                st.p[0].done = 1;
            }
        }
    } else if constexpr (MASS) {
        if (level == 0) {
            f = st.p[0];
            if (!f.done) {
                finish_k<DT>(g, r, st, waves_u, &pick, k_thr, k_ties);
                if (part == 0 && tid == 0) {
                    st.k_thr = k_thr;
                    st.k_ties = k_ties;
                }
            }
        } else {
            k_thr = st.k_thr;
            k_ties = st.k_ties;
            uint64_t have;
            f = after_p<DT, OPACITY>(a, g, r, level - 1, st.p[level - 1], st, k_thr, k_ties, waves_m, &pick_m,
                                     &have);
        }
    } else {
        f = after_k<DT>(g, r, level - 1, st.k[level - 1], waves_u, &pick);
    }
    if (level > 0 && part == 0 && tid == 0) {
        if constexpr (MASS) {
            st.p[level] = f;
        } else {
            st.k[level] = f;
            if (listed) st.k[level].done = 1;
        }
    }
    if constexpr (!MASS) {
        if (listed) {
            // a wave's load is a run of the list, its entries in order; a batch's runs stand together, the batches as they
            // came (a place asked for by every wave: 16 000 atomics on few lines, 65 us for 64 rows)
            const int lane = tid & 63, wave = tid >> 6;
            const uint32_t least = max(f.found, 1u);
            for (int64_t i0 = first; i0 < n; i0 += (int64_t)parts * kBatch * step) {
                if (i0 != first) {
#pragma unroll
                    for (int q = 0; q < kBatch; q++) keys_at<DT>(row, i0 + (int64_t)tid * kVec<DT> + q * step, n, k[q]);
                }
                uint32_t in[kBatch], upto[kBatch], all[kBatch];
#pragma unroll
                for (int q = 0; q < kBatch; q++) {
                    in[q] = 0;
#pragma unroll
                    for (int e = 0; e < kVec<DT>; e++) in[q] |= k[q][e] >= least ? 1u << e : 0u;
                    upto[q] = wave_scan((uint32_t)__builtin_popcount(in[q]));
                    all[q] = (uint32_t)__builtin_amdgcn_readlane((int)upto[q], 63);
                    if (lane == 0) waves_i[q * (kHistThreads / 64) + wave] = all[q];
                }
                __syncthreads();
                static_assert(kHistThreads / 64 * kBatch <= 64, "a lane each");
                const uint32_t one = lane < kHistThreads / 64 * kBatch ? waves_i[lane] : 0u, to_one = wave_scan(one);
                if (tid == 63 && to_one) list_at = atomicAdd(&g.list_count[(size_t)r * kListPitch], to_one);
                __syncthreads();
                const uint32_t place = list_at + to_one - one;
#pragma unroll
                for (int q = 0; q < kBatch; q++) {
                    const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)place, q * (kHistThreads / 64) + wave);
                    if (all[q] == 0) continue;
                    const int64_t i = i0 + q * step + (int64_t)tid * kVec<DT>;
                    if (lane == 0) g.list_runs[(size_t)r * g.run_pitch + i / kWaveEntries<DT>] = at | all[q] << 16;
                    uint32_t to = at + upto[q] - __builtin_popcount(in[q]);
#pragma unroll
                    for (int e = 0; e < kVec<DT>; e++)
                        if ((in[q] >> e) & 1u) g.list[(size_t)r * kListMax + to++] = make_uint2(k[q][e], (uint32_t)(i + e));
                }
            }
            return;
        }
    }
    if (f.done) return;
    const bool final_level = level == kUsedLevels<DT> - 1;
    if (!first_launch) s = st.scale;
    // Where few entries agree, a wave would compute a weight for a lane or two of every 64: they are queued (in the space
    // of the copies, which such a histogram does without), and taken 64 at a time.
    const bool queued = MASS && (level > 0 || k_thr != 0);
    const int copies = (MASS && !queued) ? kCopies : 1;
    for (int b = tid; b < kBins; b += kHistThreads) {
        if constexpr (MASS)
            for (int c = 0; c < 2 * copies; c++) mass[c * kBins + b] = 0;
        count[b] = 0;
    }
    __syncthreads();
    const int lane = tid & 63, copy = lane & (copies - 1);
    auto add = [&](uint32_t key) {
        const uint32_t d = digit_of(key, level);
        if constexpr (MASS) {
            const Words v = words_of(weight<DT, OPACITY>(key, s), a.high);
            atomicAdd((unsigned long long *)&mass[d * copies + copy], (unsigned long long)v.hi);
            atomicAdd((unsigned long long *)&mass[(d + kBins) * copies + copy], (unsigned long long)v.lo);
            if (final_level) atomicAdd(&count[d], 1u);
        } else {
            atomicAdd(&count[d], 1u);
        }
    };
    static_assert(63 + 64 * 8 <= kQueue, "a load's keys and a rest");
    uint32_t *wave_queue = reinterpret_cast<uint32_t *>(mass + (MASS ? 2 * kBins : 0)) + (tid >> 6) * kQueue;
    int waiting = 0;
    for (int64_t i0 = first; i0 < n; i0 += (int64_t)parts * kBatch * step) {
        if (i0 != first) {
#pragma unroll
            for (int q = 0; q < kBatch; q++) keys_at<DT>(row, i0 + (int64_t)tid * kVec<DT> + q * step, n, k[q]);
        }
#pragma unroll
        for (int q = 0; q < kBatch; q++) {
            uint32_t in = 0;
#pragma unroll
            for (int e = 0; e < kVec<DT>; e++)
                in |= (k[q][e] > k_thr && agrees(k[q][e], f.found, level)) ? 1u << e : 0u;
            if (!queued) {
#pragma unroll
                for (int e = 0; e < kVec<DT>; e++)
                    if ((in >> e) & 1u) add(k[q][e]);
                continue;
            }
            const uint32_t mine = __builtin_popcount(in), upto = wave_scan(mine);
            int at = waiting + (int)(upto - mine);
#pragma unroll
            for (int e = 0; e < kVec<DT>; e++)
                if ((in >> e) & 1u) wave_queue[at++] = k[q][e];
            waiting += __builtin_amdgcn_readlane((int)upto, 63);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            while (waiting >= 64) {
                waiting -= 64;
                add(wave_queue[waiting + lane]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
    if (queued) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (lane < waiting) add(wave_queue[lane]);
    }
    __syncthreads();
    for (int b = tid; b < kBins; b += kHistThreads) {
        if constexpr (MASS) {
            uint64_t hi = 0, lo = 0;
            for (int c = 0; c < copies; c++) {
                hi += mass[b * copies + c];
                lo += mass[(b + kBins) * copies + c];
            }
            unsigned long long *out = (unsigned long long *)g.p_mass + ((size_t)r * kLevels + level) * 2 * kBins + b;
            if (hi) atomicAdd(out, (unsigned long long)hi);
            if (lo) atomicAdd(out + kBins, (unsigned long long)lo);
            if (final_level && count[b]) atomicAdd(&g.p_count[(size_t)r * kBins + b], count[b]);
        } else {
            if (count[b]) atomicAdd(&g.k_count[((size_t)r * kLevels + level) * kBins + b], count[b]);
        }
    }
}

// One workgroup per row that has a list: its runs put in order, then the rest as for a short row.
template <int DT, bool OPACITY>
__global__ void __launch_bounds__(kListThreads)
k_long_list(SampleArgs a, LongArgs g, const float *__restrict__ uniforms, int32_t *__restrict__ ids) {
    __shared__ RowShared<kListThreads> sh;
    static_assert((kRunMax + kListMax) * 4 <= sizeof(sh.masses), "runs and keys in the masses' space");
    const int r = blockIdx.x, tid = threadIdx.x;
    const LongRow &st = g.rows[r];
    const int n = (int)st.listed;
    if (n == 0) return;
    int32_t *shift = reinterpret_cast<int32_t *>(sh.masses);   // of a run's entries, from the list to the order
    uint32_t *keys = reinterpret_cast<uint32_t *>(sh.masses) + kRunMax;
    const uint2 *list = g.list + (size_t)r * kListMax;
    int32_t *order = g.list_index + (size_t)r * kListMax;
    uint32_t before = 0;
    for (int i = tid; i - tid < g.run_pitch; i += kListThreads) {
        const uint32_t run = i < g.run_pitch ? g.list_runs[(size_t)r * g.run_pitch + i] : 0u;
        uint32_t all;
        const uint32_t start = before + block_scan<kListThreads>(run >> 16, sh.waves_i, all);
        if (i < g.run_pitch) shift[i] = (int32_t)start - (int32_t)(run & 0xffffu);
        before += all;
    }
    __syncthreads();
    for (int i = tid; i < kListMax; i += kListThreads) {
        if (i < n) {
            const uint2 e = list[i];
            const int at = i + shift[e.y / kWaveEntries<DT>];
            keys[at] = e.x;
            order[at] = (int32_t)e.y;
        } else {
            keys[i] = 0;
        }
    }
    __syncthreads();
    uint32_t key[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) key[e] = keys[tid * kEach + e];
    __syncthreads();
    draw_row<DT, OPACITY, kListThreads>(a, row_settings(a, r), r, key, st.scale.top, st.k[0], 1, 0, 1, sh, uniforms,
                                        ids,
                                        [&](int i) { return order[i]; });
}

// One workgroup per row: threshold and ties, once all digits are counted.
template <int DT, bool OPACITY>
__global__ void __launch_bounds__(kHistThreads)
k_long_cut(SampleArgs a, LongArgs g) {
    __shared__ uint64_t waves_u[kHistThreads / 64];
    __shared__ Mass waves_m[kHistThreads / 64];
    __shared__ Picked pick;
    __shared__ PickedOf<Mass> pick_m;
    const int r = blockIdx.x;
    LongRow &st = g.rows[r];
    constexpr int last = kUsedLevels<DT> - 1;
    if (st.listed) return;
    uint32_t thr = 0, ties = 0;
    if (g.with_p && !st.p[0].done) {
        thr = st.k_thr;
        ties = st.k_ties;
        uint64_t have = 0;
        const MassSearch f = after_p<DT, OPACITY>(a, g, r, last, st.p[last], st, thr, ties, waves_m, &pick_m, &have);
        if (!f.done) {
            thr = f.found;
            ties = ties_for(f.above, f.goal, mass_of(words_of(weight<DT, OPACITY>(thr, st.scale), a.high), a.bits), have);
        }
    } else {
        finish_k<DT>(g, r, st, waves_u, &pick, thr, ties);
    }
    if (threadIdx.x == 0) {
        st.thr = thr;
        st.ties = ties;
        st.tie_weight = 0;
        if (thr) {
            const double w = weight<DT, OPACITY>(thr, st.scale);
            st.tie_weight = w >= st.min_p ? mass_of(words_of(w, a.high), a.bits) : (Mass)0;
        }
    }
}

// Per chunk: running sums of the kept weights and of the ties per 8 entries, and their totals.  CUT false: no row has a
// threshold, and (BEGUN false) no launch has prepared the rows' state: the row's maximum is taken from its chunks' here.
template <int DT, bool OPACITY, bool CUT, bool BEGUN>
__global__ void __launch_bounds__(kChunkThreads)
k_long_sums(SampleArgs a, LongArgs g) {
    __shared__ Mass waves_m[kChunkThreads / 64];
    __shared__ uint32_t waves_i[kChunkThreads / 64];
    __shared__ uint32_t keys[CUT ? kSeg : 1][kChunkThreads];
    const int r = blockIdx.x / g.chunks, c = blockIdx.x - r * g.chunks, tid = threadIdx.x;
    if (CUT && g.rows[r].listed) return;
    const char *row = row_base<DT>(a, r);
    const int64_t i0 = (int64_t)c * kChunk + (int64_t)tid * kSeg;
    uint32_t key[kSeg];
#pragma unroll
    for (int q = 0; q < kSeg / kVec<DT>; q++) {
        uint32_t k[kVec<DT>];
        keys_at<DT>(row, i0 + q * kVec<DT>, a.cols, k);
#pragma unroll
        for (int e = 0; e < kVec<DT>; e++) key[q * kVec<DT> + e] = k[e];
    }
    uint32_t thr = 0;
    double min_p;
    Scale s;
    bool greedy, ok;
    Mass tie_weight = 0;
    if constexpr (BEGUN) {
        const LongRow &st = g.rows[r];
        thr = CUT ? st.thr : 0u;
        tie_weight = CUT ? st.tie_weight : (Mass)0;
        s = st.scale;
        min_p = st.min_p;
        greedy = st.greedy;
        ok = st.ok;
    } else {
        const LongRow st = long_row<DT, OPACITY>(a, r, row_max<kChunkThreads>(g, r, waves_i));
        s = st.scale;
        min_p = st.min_p;
        greedy = st.greedy;
        ok = st.ok;
        if (c == 0 && tid == 0) g.rows[r] = st;
    }
    Words some = {0, 0};
    auto add = [&](double w) {
        const Words v = words_of(w, a.high);
        some.hi += v.hi;
        some.lo += v.lo;
    };
    uint32_t ties = 0;
    if (ok) {
        uint32_t above = 0;
#pragma unroll
        for (int e = 0; e < kSeg; e++) {
            if (CUT && thr) ties += key[e] == thr;
            above |= (key[e] > thr && (!greedy || key[e] == s.top)) ? 1u << e : 0u;
        }
        if constexpr (CUT) {
            // A lane goes through its own kept entries: behind a cut a wave takes as many rounds as its fullest lane has,
            // not eight with a few lanes each.
#pragma unroll
            for (int e = 0; e < kSeg; e++) keys[e][tid] = key[e];
            while (above) {
                const int e = __builtin_ctz(above);
                above &= above - 1;
                const double w = weight<DT, OPACITY>(keys[e][tid], s);
                if (w >= min_p) add(w);
            }
        } else {
#pragma unroll
            for (int e = 0; e < kSeg; e++) {
                const double w = weight<DT, OPACITY>(key[e], s);
                if (((above >> e) & 1u) && w >= min_p) add(w);
            }
        }
    }
    Mass sum = mass_of(some, a.bits);
    if constexpr (CUT) {                       // (as if all ties were kept: see ChunkView)
        sum += tie_weight * ties;
    }
    const size_t at = (size_t)r * g.chunks + c, seg = at * kChunkSegs + tid;
    Mass total;
    const Mass before = block_scan<kChunkThreads>(sum, waves_m, total);
    g.seg_sum[seg] = before;
    if ((tid & 7) == 0) g.mid_sum[at * (kChunkSegs / 8) + (tid >> 3)] = before;
    if ((tid & 63) == 0) g.top_sum[at * (kChunkSegs / 64) + (tid >> 6)] = before;
    if (tid == 0) g.chunk_sum[at] = total;
    if constexpr (CUT) {
        if (thr) {
            uint32_t all;
            g.seg_ties[seg] = block_scan<kChunkThreads>(ties, waves_i, all);
            if (tid == 0) g.chunk_ties[at] = all;
        }
    }
}

// One workgroup per row: running sums over the chunks.
template <bool CUT>
__global__ void __launch_bounds__(kHistThreads)
k_long_scan(LongArgs g) {
    __shared__ Mass waves_m[kHistThreads / 64];
    __shared__ uint32_t waves_i[kHistThreads / 64];
    const int r = blockIdx.x, tid = threadIdx.x;
    LongRow &st = g.rows[r];
    if (CUT && st.listed) return;
    const size_t first = (size_t)r * g.chunks;
    const bool ok = st.ok;
    const uint32_t thr = CUT ? st.thr : 0u, ties = CUT ? st.ties : 0u;
    const Mass tie_weight = CUT ? st.tie_weight : (Mass)0;
    Mass base = 0;
    uint32_t tie_base = 0;
    for (int c0 = 0; c0 < g.chunks; c0 += kHistThreads) {
        const int c = c0 + tid;
        const bool in = c < g.chunks;
        Mass v = in ? g.chunk_sum[first + c] : (Mass)0;
        if (CUT && thr) {
            const uint32_t here = in ? g.chunk_ties[first + c] : 0u;
            uint32_t all;
            const uint32_t before = tie_base + block_scan<kHistThreads>(here, waves_i, all);
            tie_base += all;
            if (in) g.chunk_ties[first + c] = before;
            const uint32_t left = ties > before ? ties - before : 0u;
            if (left < here) v -= tie_weight * (here - left);
        }
        Mass all;
        const Mass before = base + block_scan<kHistThreads>(v, waves_m, all);
        base += all;
        if (in) g.chunk_sum[first + c] = before;
    }
    if (tid == 0) st.total = ok ? base : (Mass)0;
}

// A draw is made by LANES neighbouring lanes.  The last of `n` non-decreasing values f(0) = 0, f(1), ... that does not
// exceed `goal`, LANES values at a time; each of the lanes gets it, and its value.
template <int LANES>
static __device__ __forceinline__ uint64_t group_ballot(bool b) {
    const uint64_t m = __builtin_amdgcn_ballot_w64(b) >> (threadIdx.x & 63 & ~(LANES - 1));
    return LANES == 64 ? m : m & ((1ull << (LANES & 63)) - 1ull);
}
template <int LANES, typename F>
static __device__ __forceinline__ int last_not_above(int n, Mass goal, F f, Mass &value) {
    const int lane = threadIdx.x & (LANES - 1);
    int lo = 0;
    value = 0;
    while (n > 1) {                            // (n is the same in every lane of the wave)
        const int step = (n + LANES - 1) / LANES, at = lane * step;
        const Mass v = at < n ? f(lo + at, step) : ~(Mass)0;
        const int c = __builtin_popcountll(group_ballot<LANES>(v <= goal)) - 1;   // (f(lo) <= goal)
        value = shuffle(v, (threadIdx.x & 63 & ~(LANES - 1)) + c);
        lo += c * step;
        n = step;
    }
    return lo;
}

// A chunk's running sums as the draws see them.  The stored ones hold all of the chunk's ties; where not all are kept, the
// ones behind the `left` first are taken off.
template <bool CUT>
struct ChunkView {
    const Mass *seg_sum, *mid_sum, *top_sum;
    const uint32_t *seg_ties;
    Mass tie_weight;
    uint32_t thr, left;
    bool cut;
    __device__ ChunkView(const LongArgs &g, const LongRow &st, size_t chunk, uint32_t left_, bool cut_) {
        set(g, st, chunk);
        left = left_;
        cut = cut_;
    }
    __device__ ChunkView(const LongArgs &g, const LongRow &st, int r, int c) {
        const size_t chunk = (size_t)r * g.chunks + c;
        set(g, st, chunk);
        left = 0xffffffffu;
        cut = false;
        if (CUT && thr) {
            const uint32_t before = g.chunk_ties[chunk];
            left = st.ties > before ? st.ties - before : 0u;
            cut = c + 1 == g.chunks || g.chunk_ties[chunk + 1] - before > left;
        }
    }
    __device__ void set(const LongArgs &g, const LongRow &st, size_t chunk) {
        seg_sum = g.seg_sum + chunk * kChunkSegs;
        mid_sum = g.mid_sum + chunk * (kChunkSegs / 8);
        top_sum = g.top_sum + chunk * (kChunkSegs / 64);
        seg_ties = g.seg_ties + chunk * kChunkSegs;
        thr = CUT ? st.thr : 0u;
        tie_weight = (CUT && thr) ? st.tie_weight : (Mass)0;
    }
    // (i a multiple of `step`: neighbours of a step lie side by side, a draw touches a line per step)
    __device__ Mass sum_before(int i, int step) const {
        Mass v = step == 64 ? top_sum[i >> 6] : (step == 8 ? mid_sum[i >> 3] : seg_sum[i]);
        if (CUT && cut) {
            const uint32_t t = seg_ties[i];
            if (t > left) v -= tie_weight * (t - left);
        }
        return v;
    }
};

// A draw: the last chunk, then the last 8 entries, whose running sum does not exceed the goal, then these side by side.
// (Integer sums: what is found there holds a weight.)  Bound by the latency of some ten dependent loads, which the other
// draws' hide: eight lanes a draw make 31 000 waves of 250 000 draws, where a thread a draw left four to a SIMD and
// fetched fifteen lines (with sums of one word 50 000 draws 9.6 -> 6.7 us, 250 000 28.5 -> 26.0; of two 7.8 and 31).
// A workgroup's draws are of one row, so that what a row has in common stays in scalar registers.
template <int LANES>
constexpr int kDrawThreads = LANES == 64 ? 64 : 256;
template <int DT, bool OPACITY, bool CUT, int LANES, bool SCANNED>
__global__ void __launch_bounds__(kDrawThreads<LANES>)
k_long_draw(SampleArgs a, LongArgs g, int blocks, const float *__restrict__ uniforms, int32_t *__restrict__ ids) {
    const int r = blockIdx.x / blocks, lane = threadIdx.x & (LANES - 1);
    const int mine = (blockIdx.x - r * blocks) * (kDrawThreads<LANES> / LANES) + threadIdx.x / LANES;
    // (lanes without a draw repeat the last: a wave's steps are in common)
    const size_t at = (size_t)r * a.draws + min(mine, a.draws - 1);
    const LongRow &st = g.rows[r];
    if (CUT && st.listed) return;
    const float u = uniforms[at];
    const bool greedy = st.greedy;
    Mass total, before, rest;
    int lo;
    uint32_t left = 0xffffffffu;
    bool cut = false;
    if constexpr (SCANNED) {
        total = st.total;
        rest = (greedy || total == 0 || isnan(u)) ? (Mass)0 : goal_of(u, total);
        const Mass *chunk_sum = g.chunk_sum + (size_t)r * g.chunks;
        lo = last_not_above<LANES>(g.chunks, rest, [&](int i, int) { return i < g.chunks ? chunk_sum[i] : ~(Mass)0; }, before);
        rest -= before;
    } else {
        // up to 64 chunks, whose sums no launch has scanned: a lane each
        static_assert(SCANNED || LANES == 64, "a wave");
        const size_t chunk = (size_t)r * g.chunks + lane;
        const bool in = lane < g.chunks;
        Mass v = in ? g.chunk_sum[chunk] : (Mass)0;
        uint32_t chunk_left = 0xffffffffu, here = 0;
        if (CUT && st.thr) {
            here = in ? g.chunk_ties[chunk] : 0u;
            const uint32_t ties_before = wave_scan(here) - here;
            chunk_left = st.ties > ties_before ? st.ties - ties_before : 0u;
            if (chunk_left < here) v -= st.tie_weight * (here - chunk_left);
        }
        const Mass upto = wave_scan(v);
        total = st.ok ? shuffle(upto, 63) : (Mass)0;
        rest = (greedy || total == 0 || isnan(u)) ? (Mass)0 : goal_of(u, total);
        lo = max(__builtin_popcountll(__builtin_amdgcn_ballot_w64(in && upto - v <= rest)) - 1, 0);
        rest -= shuffle(upto - v, lo);
        left = (uint32_t)__shfl((int)chunk_left, lo, 64);
        cut = __shfl((int)(chunk_left < here), lo, 64) != 0;
    }
    const bool none = total == 0 || isnan(u);
    const ChunkView<CUT> v = SCANNED ? ChunkView<CUT>(g, st, r, lo)
                                     : ChunkView<CUT>(g, st, (size_t)r * g.chunks + lo, left, cut);
    const int seg = last_not_above<LANES>(kChunkSegs, rest, [&](int i, int step) { return v.sum_before(i, step); }, before);
    const int64_t i0 = (int64_t)lo * kChunk + (int64_t)seg * kSeg;
    uint32_t key = 0;
    if (lane < kSeg && i0 + lane < a.cols) key = key_at<DT>(row_base<DT>(a, r), i0 + lane);
    const bool tied = CUT && v.thr != 0 && key == v.thr;
    uint32_t rank = 0;                         // (where nothing is cut, every rank is below `left`)
    if (CUT && v.cut) rank = v.seg_ties[seg];
    rank += __builtin_popcountll(group_ballot<LANES>(tied) & ((1ull << lane) - 1ull));
    Mass run = 0;
    if ((key > v.thr || (tied && rank < v.left)) && (!greedy || key == st.scale.top)) {
        const double w = weight<DT, OPACITY>(key, st.scale);
        if (w >= st.min_p) run = mass_of(words_of(w, a.high), a.bits);
    }
#pragma unroll
    for (int off = 1; off < kSeg; off <<= 1) {
        const Mass o = shuffle(run, (threadIdx.x - off) & 63);
        if (lane >= off) run += o;
    }
    const uint64_t over = group_ballot<LANES>(lane < kSeg && before + run > rest);
    if (lane == 0 && mine < a.draws) ids[at] = (none || over == 0) ? -1 : (int32_t)(i0 + __builtin_ctzll(over));
}

// ---- host -------------------------------------------------------------------------------------------------------------
// Longest row of the one-workgroup form, what 1024 threads hold in registers.  Calls of 8192 entries with top-p, so / in the
// longer rows' launches: 1 row 13.5 / 39 us, 256 rows 14.2 / 56, 1024 rows 52 / 148; with nothing cut 9.0 / 15.6 and 28 / 31.
constexpr int kRowLimit = 8192;

struct SampleLayout {
    size_t rows, k_count, p_mass, p_count, chunk_max, chunk_sum, chunk_ties, seg_sum, mid_sum, top_sum, seg_ties, list, list_index,
        list_runs, list_count, total;
    int chunks, run_pitch;
    SampleLayout(int n_rows, int cols) {
        size_t o = 0;
        auto take = [&](size_t bytes) { size_t r = o; o += (bytes + 255) & ~(size_t)255; return r; };
        chunks = cols > kRowLimit ? (int)(((int64_t)cols + kChunk - 1) / kChunk) : 0;
        const size_t n = (size_t)n_rows * chunks, some = chunks ? (size_t)n_rows : 0;
        rows = take(some * sizeof(LongRow));
        k_count = take(some * kLevels * kBins * 4);
        p_mass = take(some * kLevels * 2 * kBins * 8);
        p_count = take(some * kBins * 4);
        chunk_max = take(n * 4);
        chunk_sum = take(n * sizeof(Mass));
        chunk_ties = take(n * 4);
        seg_sum = take(n * kChunkSegs * sizeof(Mass));
        mid_sum = take(n * kChunkSegs / 8 * sizeof(Mass));
        top_sum = take(n * kChunkSegs / 64 * sizeof(Mass));
        seg_ties = take(n * kChunkSegs * 4);
        run_pitch = chunks ? (int)min(((int64_t)cols + kRun - 1) / kRun, (int64_t)kRunMax) : 0;
        list = take(some * kListMax * 8);
        list_index = take(some * kListMax * 4);
        list_runs = take(some * run_pitch * 4);
        list_count = take(some * kListPitch * 4);
        total = o > 0 ? o : 256;
    }
};

// Eight draws a thread pay for a selection of one's own, as long as all the workgroups are resident at once.  With top-p, one
// workgroup a row / so: 1 x 8160, 16 384 draws 40 / 27 us, 1 M 1742 / 29; 1 x 28, 1024 draws 32 / 26, 100 000 1316 / 27;
// 2000 x 28 (more rows than are resident) would go from 111 to 198 with two a row.
template <int DT, bool OPACITY, int THREADS>
static int launch_row_form(const SampleArgs &a, const float *uniforms, int32_t *ids, hipStream_t s) {
    const int64_t room = 256 * (160 * 1024 / (int64_t)sizeof(RowShared<THREADS>)) / a.rows, share = 8 * THREADS;
    int64_t parts = ((int64_t)a.draws + share - 1) / share;
    parts = parts < room ? parts : (room < 1 ? 1 : room);
    GS_LAUNCH((k_sample_row<DT, OPACITY, THREADS>), dim3((unsigned)(parts * a.rows)), dim3(THREADS), 0, s, a, (int)parts, uniforms,
              ids);
    GS_LAUNCH_CHECK();
    return GS_OK;
}
template <int DT, bool OPACITY>
static int launch_rows(const SampleArgs &a, const float *uniforms, int32_t *ids, hipStream_t s) {
    if (a.cols <= 64 * kEach) return launch_row_form<DT, OPACITY, 64>(a, uniforms, ids, s);
    if (a.cols <= 256 * kEach) return launch_row_form<DT, OPACITY, 256>(a, uniforms, ids, s);
    return launch_row_form<DT, OPACITY, 1024>(a, uniforms, ids, s);
}

// Up to this many chunks (8 M entries) the launch behind k_long_max reads the chunks' maxima itself, a few loads a thread;
// beyond, that would grow with the square of the row.  Rows with nothing cut, in a launch of its own / in the next one:
// 1 M 22.2 / 18.7 us a call, 5 M 29.6 / 28.3, 16 M 56 / 62, 40 M 113 / 140.
constexpr int kOwnMaxChunks = 2048;

// Up to this many draws a wave each, in fewer steps and without a scan's launch for short rows.  Calls of 64 x 131072 with
// nothing cut, a wave / eight lanes a draw: 64 draws 30.4 / 33.3 us, 2048 31.1 / 33.4, 16 384 37.4 / 34.5.
constexpr int64_t kWaveDraws = 2048;

template <int DT, bool OPACITY, bool CUT>
static int launch_long(const SampleArgs &a, LongArgs g, const float *uniforms, int32_t *ids, hipStream_t s) {
    const dim3 chunks((unsigned)((int64_t)a.rows * g.chunks)), rows(a.rows);
    // two workgroups per compute unit over all the rows, none without a batch of loads
    const int64_t batch = (int64_t)kHistThreads * kVec<DT> * kBatch, most = ((int64_t)a.cols + batch - 1) / batch;
    int64_t parts = (512 + a.rows - 1) / a.rows;
    if (parts > most) parts = most;
    const dim3 grid((unsigned)(parts * a.rows));
    // One for the masses: every workgroup adds its two words of up to 2048 bins to the row's (calls of 5 M opacities and of
    // 64 x 131072 with top-p: 256 workgroups 116 and 81 us, 512 for the first digit 119 and 83, for all of them 135 and 102,
    // 128 behind the first 129 and 98)
    const int64_t fewer = (256 + a.rows - 1) / a.rows, mass_parts = fewer < parts ? fewer : parts;
    const bool with_k = CUT && g.with_k, begun = !with_k && g.chunks > kOwnMaxChunks;
    if (with_k) {
        g.maxima = (int)parts;                 // (a batch is at least a chunk)
        const int some = parts < 4 ? (int)parts : 4;
        GS_LAUNCH((k_long_empty<DT>), dim3((unsigned)(some * a.rows)), dim3(kHistThreads), 0, s, g, some);
        GS_LAUNCH_CHECK();
        GS_LAUNCH((k_long_first<DT>), grid, dim3(kHistThreads), 0, s, a, g, (int)parts);
    } else {
        GS_LAUNCH((k_long_max<DT>), chunks, dim3(kChunkThreads), 0, s, a, g);
    }
    GS_LAUNCH_CHECK();
    if (begun) {
        GS_LAUNCH((k_long_begin<DT, OPACITY>), rows, dim3(kHistThreads), 0, s, a, g);
        GS_LAUNCH_CHECK();
    }
    if constexpr (CUT) {
        if (with_k) {
            for (int level = 1; level < kUsedLevels<DT>; level++) {
                GS_LAUNCH((k_long_digit<DT, OPACITY, false>), grid, dim3(kHistThreads), 0, s, a, g, (int)parts, level,
                          level == 1);
                GS_LAUNCH_CHECK();
                if (level == 1 && g.lists) {
                    GS_LAUNCH((k_long_list<DT, OPACITY>), rows, dim3(kListThreads), 0, s, a, g, uniforms, ids);
                    GS_LAUNCH_CHECK();
                }
            }
        }
        if (g.with_p)
            for (int level = 0; level < kUsedLevels<DT>; level++) {
                GS_LAUNCH((k_long_digit<DT, OPACITY, true>), dim3((unsigned)(mass_parts * a.rows)), dim3(kHistThreads), 0, s, a, g,
                          (int)mass_parts, level, !begun && !with_k && level == 0);
                GS_LAUNCH_CHECK();
            }
        GS_LAUNCH((k_long_cut<DT, OPACITY>), rows, dim3(kHistThreads), 0, s, a, g);
        GS_LAUNCH_CHECK();
    }
    if (CUT || begun) {
        GS_LAUNCH((k_long_sums<DT, OPACITY, CUT, true>), chunks, dim3(kChunkThreads), 0, s, a, g);
    } else {
        GS_LAUNCH((k_long_sums<DT, OPACITY, false, false>), chunks, dim3(kChunkThreads), 0, s, a, g);
    }
    GS_LAUNCH_CHECK();
    const bool few = (int64_t)a.rows * a.draws <= kWaveDraws;
    const bool scanned = !few || g.chunks > 64;
    if (scanned) {
        GS_LAUNCH((k_long_scan<CUT>), rows, dim3(kHistThreads), 0, s, g);
        GS_LAUNCH_CHECK();
    }
    if (!scanned) {
        GS_LAUNCH((k_long_draw<DT, OPACITY, CUT, 64, false>), dim3((unsigned)(a.rows * a.draws)), dim3(64), 0, s, a, g,
                  a.draws, uniforms, ids);
    } else if (few) {
        GS_LAUNCH((k_long_draw<DT, OPACITY, CUT, 64, true>), dim3((unsigned)(a.rows * a.draws)), dim3(64), 0, s, a, g,
                  a.draws, uniforms, ids);
    } else {
        const int blocks = (int)(((int64_t)a.draws + 31) / 32);
        GS_LAUNCH((k_long_draw<DT, OPACITY, CUT, 8, true>), dim3((unsigned)((int64_t)blocks * a.rows)), dim3(256), 0, s, a, g,
                  blocks, uniforms, ids);
    }
    GS_LAUNCH_CHECK();
    return GS_OK;
}

template <int DT, bool OPACITY>
static int launch_sample(const SampleArgs &a, const float *uniforms, int32_t *ids, char *ws, const SampleLayout &L,
                         hipStream_t s) {
    if (L.chunks == 0) return launch_rows<DT, OPACITY>(a, uniforms, ids, s);
    const GsSampleConfig &c = a.cfg;
    const bool with_k = c.top_k_rows || c.top_k > 0, with_p = c.top_p_rows || c.top_p < 1.0f;
    // Not for a k that no list can hold, where the host knows it, for rows of more runs than a workgroup's table has, or for
    // more draws than one workgroup a row should make (1.4 us a thousand, where the whole chip makes a thousand draws of all
    // the rows in 0.08; a list saves some 10 us of passes).  1 x 20000, top-k 4000: 4096 draws 45 us listed, 39 not, 32 768
    // 82 and 40, 131 072 226 and 45; 16 x 1 M: 16 384 draws 81 and 97, 131 072 264 and 225; 64 x 131072: 32 768 119 and 218.
    const bool lists = with_k && (c.top_k_rows || c.top_k <= kListMax) && a.cols <= (int64_t)kRunMax * kWaveEntries<DT> &&
                       (int64_t)a.draws * (18 - a.rows) <= 18 * 4096;
    const LongArgs g = {(LongRow *)(ws + L.rows), (uint32_t *)(ws + L.k_count), (uint64_t *)(ws + L.p_mass),
                        (uint32_t *)(ws + L.p_count), (uint32_t *)(ws + L.chunk_max), (Mass *)(ws + L.chunk_sum),
                        (uint32_t *)(ws + L.chunk_ties), (Mass *)(ws + L.seg_sum), (Mass *)(ws + L.mid_sum),
                        (Mass *)(ws + L.top_sum), (uint32_t *)(ws + L.seg_ties),
                        (uint2 *)(ws + L.list), (int32_t *)(ws + L.list_index), (uint32_t *)(ws + L.list_runs),
                        (uint32_t *)(ws + L.list_count), L.chunks, L.chunks, L.run_pitch, with_k, with_p, lists};
    return with_k || with_p ? launch_long<DT, OPACITY, true>(a, g, uniforms, ids, s)
                            : launch_long<DT, OPACITY, false>(a, g, uniforms, ids, s);
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
    const SampleLayout L(rows, cols);
    // a launch's threads, 32 bits
    const int64_t row_threads = cols <= 64 * kEach ? 64 : (cols <= 256 * kEach ? 256 : 1024);
    const int64_t most = L.chunks == 0 ? rows * row_threads
                                       : (int64_t)rows * (L.chunks > kHistThreads / kChunkThreads ? (int64_t)L.chunks * kChunkThreads
                                                                                                  : (int64_t)kHistThreads);
    if (most > 0xffffffffLL ||
        (L.chunks && (int64_t)rows * (((int64_t)draws + 31) / 32) > 0xffffffffLL / 256))
        return GS_ERR_UNSUPPORTED;
    if (workspace_bytes < L.total) return GS_ERR_WORKSPACE;
    int log_cols = 12;
    while (((int64_t)1 << log_cols) < cols) log_cols++;
    const int bits = 62 - log_cols;
    // (a list holds kListMax entries at most, whatever the row's length)
    static_assert(kListMax == 8192 && kRowLimit == 8192, "sums of 2^13 weights of 2^49");
    const SampleArgs a = {logits, row_stride, rows, cols, draws, ldexp(1.0, log_cols == 12 ? 50 : 49), ldexp(1.0, bits), bits, *cfg};
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
