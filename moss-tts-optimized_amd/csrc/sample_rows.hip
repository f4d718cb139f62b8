// One index per row of logits from a given uniform number: temperature, top-k, top-p and min-p, per row.
//
// With the row's largest logit M, w_i = exp((x_i - M) / T) and the order "larger x first, equal ones by index":
//   top_k:  the first top_k entries (top_k <= 0 or >= vocab: all)
//   top_p:  of those, the ones whose predecessors' sum of w is at most top_p times the sum over all of them (>= 1: all)
//   min_p:  of those, the ones with w_i >= min_p
// All three keep a prefix of the order.  Drawn is the first kept index i, in index order, with
// sum_{j <= i, kept} w_j > u sum_kept w_j.  T <= 0: the first of the largest logits.  NaN counts as -inf; an entry of
// +inf leaves the others no weight; a row with nothing above -inf gives -1.
//
// Weights are integers, round(w 2^44): their sums have no order, so atomics and any split of a row give the same bits
// from call to call, and the error of a sum (2^-45 of the largest weight per entry) lies far under the distance between
// a border of the distribution and a uniform number, except for one draw in about 10^6.
//
// The borders of the prefix are found without sorting: a histogram (count and sum of w) over bins of 1/32 octave of w,
// then the border bin's own entries; of the entries with the border's key, the first few in index order are kept.
//
// What bounds it: the arithmetic of w in 64 bits, counting in LDS, and for few rows the chain of steps.  A row is read by
// several workgroups, in five launches (largest logit; histogram; border; weight of each segment of 512 entries; draw), of
// which the segments form w for the kept entries, and the histogram for all of a row with top-p, unless its bins are single
// values that need only be counted (bf16).  Then, for more than kFewRows rows, the counts also say which part of the row the
// drawn entry lies in, and one launch in place of the last three finds the border and reads that part alone.  w takes 14
// operations in 64 bits, of 8 cycles each for a wave.  128 rows of 151,936 bf16 logits, each with its own settings: 53 us;
// with the last three launches 61 (9 + 18 + 12 + 18 + 6), with linear bins besides 84, of those with a series of ten terms and
// no table 93, and one workgroup a row 309.  One row: 29 us with top-p, 19 without, 182 by one workgroup.  Rows without such
// bins (fp16, fp32, bf16 with a largest logit below 2^-9, as of log-probabilities) take 46, 48 and 31 us for one row with
// top-p, 95, 114 and 96 for 128.  A row of up to 2048 entries is one wave's: it holds them and their weights in registers, and
// needs no barrier (512 rows of 1024: 13.8 us, 46 before; fp32 14.6).
#include "wave_scan.h"

namespace moss {
namespace {

constexpr int kSpan = 46;                  // octaves: smaller weights are 0
constexpr int kBins = 32 * kSpan;          // 32 an octave
constexpr int kSegment = 512;              // entries
constexpr int kSmall = 2048;               // entries of a row that one wave takes
constexpr int kMaxVocab = 1 << 19;         // entries of 2^44 at most: a sum is at most 2^63
constexpr int kMaxChunks = 16;             // workgroups that read a row together

struct SampleArgs {
    const void* logits;
    long long stride;
    int vocab;
    const float* uniform;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    float temperature_v, top_p_v, min_p_v;
    int top_k_v;
    int64_t* out;
};

__device__ __forceinline__ float half_value(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits); }

// Eight logits as they are compared: NaN below everything, -0 equal to 0 (CLEAN false: as they are).
template <int TYPE, bool CLEAN = true>
__device__ __forceinline__ void unpack8(const u32x4_t* w, float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (TYPE == 2) {
            const uint32_t a = w[j / 2][2 * (j & 1)], b = w[j / 2][2 * (j & 1) + 1];
            x[2 * j] = __uint_as_float(a);
            x[2 * j + 1] = __uint_as_float(b);
        } else {
            const uint32_t word = w[0][j];
            x[2 * j] = TYPE == 0 ? bf16_lo(word) : half_value(word & 0xffffu);
            x[2 * j + 1] = TYPE == 0 ? bf16_hi(word) : half_value(word >> 16);
        }
    }
    if constexpr (CLEAN)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = x[j] != x[j] ? -INFINITY : x[j] + 0.0f;
}

// The ones from index i on; -inf behind the row's end.
template <int TYPE>
__device__ __forceinline__ void load8(const void* row, int i, int vocab, bool aligned, float (&x)[8]) {
    if (aligned && i + 8 <= vocab) {
        constexpr int W = TYPE == 2 ? 2 : 1;
        u32x4_t w[W];
#pragma unroll
        for (int k = 0; k < W; ++k) w[k] = reinterpret_cast<const u32x4_t*>(row)[(size_t)(i / 8) * W + k];
        unpack8<TYPE>(w, x);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (i + j >= vocab)
            x[j] = -INFINITY;
        else if constexpr (TYPE == 0)
            x[j] = bf16_bits(reinterpret_cast<const uint16_t*>(row)[i + j]);
        else if constexpr (TYPE == 1)
            x[j] = (float)reinterpret_cast<const _Float16*>(row)[i + j];
        else
            x[j] = reinterpret_cast<const float*>(row)[i + j];
        x[j] = x[j] != x[j] ? -INFINITY : x[j] + 0.0f;
    }
}

// Order-preserving key of a logit; neighbouring values of the type are neighbours (the low bits of an fp32 number that a
// 16-bit type does not have are left out).
template <int TYPE>
constexpr int kLowBits = TYPE == 0 ? 16 : TYPE == 1 ? 13 : 0;
template <int TYPE>
constexpr uint32_t kLowest = 0x007fffffu >> kLowBits<TYPE>;  // the key of -inf
template <int TYPE>
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u ? ~b : b | 0x80000000u) >> kLowBits<TYPE>;
}
template <int TYPE>
__device__ __forceinline__ float logit_of(uint32_t k) {
    const uint32_t b = k << kLowBits<TYPE>;
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~(b | ((1u << kLowBits<TYPE>) - 1)));
}

// One row's settings, and its largest logit once it is known.
struct Row {
    const void* at;
    int vocab;
    bool aligned;  // 16-byte loads
    float temperature, top_p, min_p;
    int top_k;
    bool by_k, by_p;
    float top;
    double rate;  // parts of 1/32 octave of w per unit of a logit: 32 log2(e) / T
};

template <int TYPE>
__device__ __forceinline__ Row row_of(const SampleArgs& a, int i) {
    Row r;
    r.at = reinterpret_cast<const unsigned char*>(a.logits) + (size_t)i * a.stride * (TYPE == 2 ? 4 : 2);
    r.vocab = a.vocab;
    r.aligned = MOSS_ALIGNED(r.at, 16);
    const float t = a.temperature ? a.temperature[i] : a.temperature_v;
    r.temperature = t > 3.4e38f ? 3.4e38f : t;  // times the distance of an entry of -inf it stays infinite
    r.top_k = a.top_k ? a.top_k[i] : a.top_k_v;
    r.top_p = a.top_p ? a.top_p[i] : a.top_p_v;
    r.min_p = fminf(a.min_p ? a.min_p[i] : a.min_p_v, 1.f);
    r.by_k = r.top_k > 0 && r.top_k < r.vocab;
    r.by_p = r.top_p < 1.f;
    return r;
}

// The largest logit with its first index, as one number whose maximum is looked for (0: none).
template <int TYPE>
__device__ __forceinline__ unsigned long long top_code(float x, int i) {
    return ((unsigned long long)key_of<TYPE>(x) << 32) | (uint32_t)~i;
}
// Sets the row's largest logit; false when there is nothing to draw (then `index` is the answer).
template <int TYPE>
__device__ __forceinline__ bool take_top(Row& r, unsigned long long code, int& index) {
    const uint32_t k = (uint32_t)(code >> 32);
    r.top = logit_of<TYPE>(k);
    index = k > kLowest<TYPE> ? (int)~(uint32_t)code : -1;
    r.rate = 32.0 * 1.4426950408889634 / (double)r.temperature;
    return k > kLowest<TYPE> && r.temperature > 0.f;
}

// Eight entries at a time from `begin` to `end`, `step` apart: fn(i, x).  N loads are on their way together.
template <int TYPE, int N, bool CLEAN = true, typename Fn>
__device__ __forceinline__ void walk(const Row& r, int begin, int end, int step, Fn fn) {
    float x[8];
    if (!r.aligned || r.vocab < 8) {
        for (int i = begin; i < end; i += step) {
            load8<TYPE>(r.at, i, r.vocab, false, x);
            fn(i, x);
        }
        return;
    }
    constexpr int W = TYPE == 2 ? 2 : 1;
    const u32x4_t* at = reinterpret_cast<const u32x4_t*>(r.at);
    const int last = r.vocab / 8 - 1;  // the last whole eight
    for (int i0 = begin; i0 < end; i0 += N * step) {
        u32x4_t raw[N][W];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < W; ++k) raw[n][k] = at[(size_t)min((i0 + n * step) / 8, last) * W + k];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = i0 + n * step;
            if (i >= end) break;
            if (i + 8 <= r.vocab) {
                unpack8<TYPE, CLEAN>(raw[n], x);
            } else {
                load8<TYPE>(r.at, i, r.vocab, false, x);
            }
            fn(i, x);
        }
    }
}

// How far a logit lies under the largest one, in parts of 1/32 octave of w: at most all of them, where the weight is 0.
// (A largest logit of +inf less itself is a NaN, which the maximum makes 0.)
__device__ __forceinline__ double parts_of(const Row& r, float x) {
    return fmin(fmax(((double)r.top - (double)x) * r.rate, 0.0), (double)kBins);
}
__device__ __forceinline__ int bin_of(double parts) { return (int)__builtin_rint(parts); }
// w 2^44, to the nearest integer: 2^(44 - q / 32) for the nearest whole q from a table of 32 and the exponent's bits, times
// the series of exp for the rest of at most 1/64 octave, off by less than 2 10^-12; adding 2^52 rounds to an integer.
__device__ __forceinline__ unsigned long long weight_at(double parts, const double* table) {
    const double n = __builtin_rint(parts), y = (n - parts) * (0.6931471805599453 / 32.0);
    const int q = (int)n;
    double p = 1.0 / 24.0;
    p = fma(p, y, 1.0 / 6.0);
    p = fma(p, y, 0.5);
    p = fma(p, y, 1.0);
    p = fma(p, y, 1.0);
    const double t = table[q & 31];
    const double power = __hiloint2double(__double2hiint(t) - ((q >> 5) << 20), __double2loint(t));
    return (unsigned long long)__double_as_longlong(fma(p, power, 4503599627370496.0)) & 0xfffffffffffffull;
}
__device__ __forceinline__ unsigned long long weight_of(const Row& r, float x, const double* table) {
    return weight_at(parts_of(r, x), table);
}
__device__ __forceinline__ void fill_table(double* table, int tid) {
    if (tid < 32) table[tid] = exp2(44.0 - tid / 32.0);
}

// The smallest key up to the largest logit's that fulfils a condition which the largest one does and, once it holds,
// holds for every larger key.  64 keys a turn; every lane gets the answer.
template <int TYPE, typename Fn>
__device__ __forceinline__ uint32_t first_key(uint32_t top, int lane, Fn holds) {
    uint32_t lo = kLowest<TYPE>, hi = top;  // it fails at lo
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + kWave - 1) / kWave;
        const uint32_t k = min(hi - lo, step * (uint32_t)(lane + 1)) + lo;
        const unsigned long long mask = __ballot(k == hi || holds(logit_of<TYPE>(k)));
        const uint32_t l = (uint32_t)__builtin_ctzll(mask);
        hi = min(hi - lo, step * (l + 1)) + lo;
        lo += l ? min(hi - lo - 1, step * l) : 0;
    }
    return hi;
}
template <int TYPE>
__device__ __forceinline__ uint32_t first_key_of_bins(const Row& r, int bin, int lane) {  // of bins 0 .. bin
    return first_key<TYPE>(key_of<TYPE>(r.top), lane, [&](float x) { return bin_of(parts_of(r, x)) <= bin; });
}
template <int TYPE>
__device__ __forceinline__ uint32_t first_key_of_min_p(const Row& r, int lane) {
    return first_key<TYPE>(key_of<TYPE>(r.top), lane, [&](float x) { return exp2(parts_of(r, x) / -32.0) >= (double)r.min_p; });
}

// The border of the prefix: entries with a key above `key` are inside, and the first `ties` with that key.
struct Border {
    uint32_t key, ties;
    unsigned long long sum;  // of the entries inside
};

// What the border looked for is: the first `need` entries, or the ones whose predecessors weigh at most `limit`.
struct Goal {
    bool by_count;
    uint32_t need;
    unsigned long long limit;
    __device__ __forceinline__ bool inside(uint32_t count, unsigned long long sum) const {
        return by_count ? count < need : sum <= limit;
    }
    // of n entries of weight w with one key, behind the given ones
    __device__ __forceinline__ Border end(uint32_t key, uint32_t n, unsigned long long w, uint32_t count,
                                          unsigned long long sum) const {
        uint32_t ties = n;
        if (by_count)
            ties = min(n, need - count);
        else if (w)
            ties = (uint32_t)min((unsigned long long)n, (limit - sum) / w + 1);
        return Border{key, ties, sum + ties * w};
    }
};
__device__ __forceinline__ unsigned long long share_limit(const Row& r, unsigned long long total) {
    return (unsigned long long)((double)fmaxf(r.top_p, 0.f) * (double)total);
}
// The number that the sums through the kept entries are held against.  u outside [0, 1) draws the first or the last kept
// entry; totals reach 2^63 (2^19 entries of full weight), and 2^64 - 2^11 is the last double that an integer holds.
__device__ __forceinline__ unsigned long long target_of(float u, unsigned long long total) {
    const double goal = (double)u * (double)total;
    return goal > 0.0 ? min((unsigned long long)fmin(goal, 18446744073709549568.0), total - 1) : 0;
}

__device__ __forceinline__ unsigned long long wave_largest(unsigned long long v) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const unsigned long long o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}
// Inclusive sum over the workgroup's threads; `parts` holds one value a wave and is free again afterwards.
template <typename V>
__device__ __forceinline__ V block_prefix(V v, V* parts, int lane, int wave) {
    v = wave_prefix(v);
    if (lane == kWave - 1) parts[wave] = v;
    __syncthreads();
    const V before = wave_prefix(lane < wave ? parts[lane] : (V)0);
    __syncthreads();
    return v + lane_value(before, kWave - 1);
}

// ---------------------------------------------------------------- long rows: several workgroups a row
// A row of bf16 logits holds few different values that matter: a bin for each from the largest logit down to 2^-9 and from
// -2^-9 down to where no weight is left, and one for what lies between.  A bin's entries weigh the same, so they need only
// be counted.  `on`: the row's values fit the bins (a largest logit of 2^-9 to 2^7, and weights that end soon enough below 0).
struct KeyBins {
    bool on;
    uint32_t top;
    int np, all;  // bin np: what lies between
};
constexpr int kKeyBins = 4096;
constexpr uint32_t kLeastPositive = 0xbb00u, kLeastNegative = 0x44ffu;  // the keys of 2^-9 and -2^-9
template <int TYPE>
__device__ __forceinline__ KeyBins key_bins(const Row& r) {
    KeyBins q{false, 0, 0, 0};
    if constexpr (TYPE == 0) {
        q.top = key_of<TYPE>(r.top);
        q.np = (int)(q.top - kLeastPositive) + 1;
        const float far = (float)((double)r.top - kBins / r.rate);  // no weight is left below; two keys to be sure
        const int kf = far > -3.3e38f ? (int)key_of<TYPE>(far) - 2 : (int)kLowest<TYPE>;
        q.all = q.np + 1 + max((int)kLeastNegative - kf, 0);
        q.on = q.top >= kLeastPositive && q.np <= kKeyBins / 2 && q.all <= kKeyBins;
    }
    return q;
}
__device__ __forceinline__ int bin_of_key(const KeyBins& q, uint32_t k) {  // q.all and more: no weight
    return k >= kLeastPositive ? (int)(q.top - k) : k > kLeastNegative ? q.np : q.np + 1 + (int)(kLeastNegative - k);
}
__device__ __forceinline__ uint32_t key_of_bin(const KeyBins& q, int b) {
    return b < q.np ? q.top - (uint32_t)b : kLeastNegative - (uint32_t)(b - q.np - 1);
}

// A chunk's bins in the workspace: sums and counts of the bins that are linear in log w, or the sum of the bin between
// and the counts of the key bins.
constexpr int kBinBytes = 12 * kBins;
static_assert(kBinBytes % 16 == 0 && kBinBytes >= 16 + 4 * kKeyBins, "a chunk's bins");
struct Work {
    unsigned long long* top;    // [rows, chunks]
    unsigned char* bins;        // [rows, chunks, kBinBytes]
    unsigned long long* seg;    // [rows, segments]: weight of the entries above the border's key
    uint32_t* tie;              // [rows, segments]: entries with the border's key
    uint2* border;              // [rows]
    int chunks, chunk, segments;  // chunk: entries, whole segments
    bool finish;                  // sample_finish_kernel draws: it wants every row's key bins
};

template <int TYPE>
__device__ __forceinline__ bool load_top(Row& r, const Work& w, int row, int lane, int& index) {
    unsigned long long c = 0;
    for (int i = lane; i < w.chunks; i += kWave) c = max(c, w.top[(size_t)row * w.chunks + i]);
    return take_top<TYPE>(r, wave_largest(c), index);
}

template <int TYPE>
__global__ __launch_bounds__(512) void sample_top_kernel(SampleArgs a, Work w) {
    __shared__ unsigned long long parts[8];
    const int row = blockIdx.x / w.chunks, chunk = blockIdx.x % w.chunks, tid = threadIdx.x, lane = tid & (kWave - 1);
    const Row r = row_of<TYPE>(a, row);
    const int end = min(r.vocab, (chunk + 1) * w.chunk);
    unsigned long long best = 0;
    walk<TYPE, 5>(r, chunk * w.chunk + 8 * tid, end, 8 * 512, [&](int i, const float(&x)[8]) {
        float m = x[0];
        int at = 0;
#pragma unroll
        for (int j = 1; j < 8; ++j)
            if (x[j] > m) m = x[j], at = j;
        best = max(best, top_code<TYPE>(m, i + at));
    });
    best = wave_largest(best);
    if (lane == 0) parts[tid / kWave] = best;
    __syncthreads();
    if (tid == 0) {
        for (int v = 0; v < 8; ++v) best = max(best, parts[v]);
        w.top[(size_t)row * w.chunks + chunk] = best;
    }
}

template <int TYPE>
__global__ __launch_bounds__(512) void sample_bins_kernel(SampleArgs a, Work w) {
    __shared__ double table[32];
    __shared__ __attribute__((aligned(16))) unsigned char bins[kBinBytes];
    const int row = blockIdx.x / w.chunks, chunk = blockIdx.x % w.chunks, tid = threadIdx.x, lane = tid & (kWave - 1);
    Row r = row_of<TYPE>(a, row);
    int index;
    if (!load_top<TYPE>(r, w, row, lane, index)) return;  // uniform
    const KeyBins q = key_bins<TYPE>(r);
    if (!(r.by_k || r.by_p || (w.finish && q.on))) return;
    fill_table(table, tid);
    const u32x4_t zero = {0u, 0u, 0u, 0u};
    for (int b = tid; b < kBinBytes / 16; b += 512) reinterpret_cast<u32x4_t*>(bins)[b] = zero;
    __syncthreads();
    unsigned long long* sum = reinterpret_cast<unsigned long long*>(bins);
    const int end = min(r.vocab, (chunk + 1) * w.chunk);
    int used = kBinBytes / 16;
    if (q.on) {
        uint32_t* count = reinterpret_cast<uint32_t*>(bins + 16);
        walk<TYPE, 5>(r, chunk * w.chunk + 8 * tid, end, 8 * 512, [&](int, const float(&x)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int b = bin_of_key(q, key_of<TYPE>(x[j]));
                // (a key above the row's largest, as when the logits change under the kernel, has no bin)
                if ((uint32_t)b < (uint32_t)q.all) atomicAdd(&count[b], 1u);
                if (b == q.np && (r.by_p || w.finish)) atomicAdd(sum, weight_of(r, x[j], table));
            }
        });
        used = 1 + (q.all + 3) / 4;
    } else {
        uint32_t* count = reinterpret_cast<uint32_t*>(bins + 8 * kBins);
        walk<TYPE, 5>(r, chunk * w.chunk + 8 * tid, end, 8 * 512, [&](int, const float(&x)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double o = parts_of(r, x[j]);
                const unsigned long long v = r.by_p ? weight_at(o, table) : 0;
                const int b = bin_of(o);
                if (b >= kBins) continue;
                if (r.by_k) atomicAdd(&count[b], 1u);
                if (r.by_p) atomicAdd(&sum[b], v);
            }
        });
    }
    __syncthreads();
    u32x4_t* to = reinterpret_cast<u32x4_t*>(w.bins + ((size_t)row * w.chunks + chunk) * kBinBytes);
    for (int b = tid; b < used; b += 512) to[b] = reinterpret_cast<const u32x4_t*>(bins)[b];
}

constexpr int kBorderThreads = 1024, kBorderWaves = kBorderThreads / kWave;
constexpr int kList = 4096;

// A bin's entries and weight, and those of everything above it.
struct Bin {
    int bin;  // -1: none
    uint32_t count, before_count;
    unsigned long long sum, before_sum;
};

struct BorderShared {
    double table[32];
    unsigned long long sum[2048];
    uint32_t count[2048];
    float list[kList];
    unsigned long long part_sum[kBorderWaves];
    uint32_t part_count[kBorderWaves];
    Bin found[kBorderWaves];
    uint32_t listed;
};

// The last bin whose first entry is inside; thread t holds bins N t .. + N - 1.  Two barriers, the first behind all that
// the caller has read of sh's bins.
template <int N>
__device__ __forceinline__ Bin border_bin(BorderShared& sh, const Goal& goal, const uint32_t (&c)[N],
                                          const unsigned long long (&s)[N], uint32_t base_count, unsigned long long base_sum) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    uint32_t ct = 0;
    unsigned long long st = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        ct += c[i];
        st += s[i];
    }
    const uint32_t cp = wave_prefix(ct);
    const unsigned long long sp = wave_prefix(st);
    if (lane == kWave - 1) {
        sh.part_count[wave] = cp;
        sh.part_sum[wave] = sp;
    }
    __syncthreads();
    uint32_t cb = base_count + wave_total(lane < wave ? sh.part_count[lane] : 0u) + cp - ct;
    unsigned long long sb = base_sum + wave_total(lane < wave ? sh.part_sum[lane] : 0ull) + sp - st;
    Bin mine{-1, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if ((c[i] || s[i]) && goal.inside(cb, sb)) mine = Bin{N * tid + i, c[i], cb, s[i], sb};
        cb += c[i];
        sb += s[i];
    }
    const unsigned long long any = __ballot(mine.bin >= 0);
    if (any ? lane == 63 - __builtin_clzll(any) : lane == 0) sh.found[wave] = mine;
    __syncthreads();
    const unsigned long long waves = __ballot(lane < kBorderWaves && sh.found[lane < kBorderWaves ? lane : 0].bin >= 0);
    return waves ? sh.found[63 - __builtin_clzll(waves)] : Bin{-1, 0, 0, 0, 0};
}

// The border inside the keys lo .. hi, which n entries have (0: not known, more than one key), behind the given ones.
// (Entries that an earlier border left out weigh on no decision: what lies before them exceeds the limit.)  Up to kList
// entries are collected first; then bins over equal parts of the keys' range, until a bin is one key.
template <int TYPE>
__device__ Border border_among(BorderShared& sh, const Row& r, const Goal& goal, uint32_t lo, uint32_t hi, uint32_t n,
                               uint32_t base_count, unsigned long long base_sum) {
    const int tid = threadIdx.x;
    bool listed = n <= kList && lo != hi;
    if (listed) {
        const float xlo = logit_of<TYPE>(lo), xhi = logit_of<TYPE>(hi);
        if (tid == 0) sh.listed = 0;
        __syncthreads();
        walk<TYPE, TYPE == 2 ? 5 : 10, false>(r, 8 * tid, r.vocab, 8 * kBorderThreads, [&](int, const float(&x)[8]) {
            uint32_t hits = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) hits |= __builtin_amdgcn_fmed3f(x[j], xlo, xhi) == x[j] ? 1u << j : 0u;
            if (!hits) return;
            uint32_t at = atomicAdd(&sh.listed, (uint32_t)__popc(hits));
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (hits >> j & 1) {
                    if (at < kList) sh.list[at] = x[j] + 0.0f;
                    ++at;
                }
        });
        __syncthreads();
        listed = sh.listed <= kList;
    }
    const int entries = listed ? (int)sh.listed : r.vocab;
    while (lo != hi) {
        const uint32_t range = hi - lo;
        const int shift = max(0, 32 - __builtin_clz(range) - 11);
        for (int b = tid; b < 2048; b += kBorderThreads) {
            sh.sum[b] = 0;
            sh.count[b] = 0;
        }
        __syncthreads();
        auto add = [&](float x) {
            const uint32_t k = key_of<TYPE>(x);
            if (k - lo > range) return;
            atomicAdd(&sh.count[(hi - k) >> shift], 1u);
            if (r.by_p) atomicAdd(&sh.sum[(hi - k) >> shift], weight_of(r, x, sh.table));
        };
        if (listed) {
            for (int i = tid; i < entries; i += kBorderThreads) add(sh.list[i]);
        } else {
            walk<TYPE, 4>(r, 8 * tid, entries, 8 * kBorderThreads, [&](int, const float(&x)[8]) {
#pragma unroll
                for (int j = 0; j < 8; ++j) add(x[j]);
            });
        }
        __syncthreads();
        const uint32_t c[2] = {sh.count[2 * tid], sh.count[2 * tid + 1]};
        const unsigned long long s[2] = {sh.sum[2 * tid], sh.sum[2 * tid + 1]};
        const Bin f = border_bin<2>(sh, goal, c, s, base_count, base_sum);
        if (f.bin < 0) return Border{kLowest<TYPE> + 1, 0xffffffffu, 0};  // only when the logits change under the kernel
        base_count = f.before_count;
        base_sum = f.before_sum;
        n = f.count;
        hi -= (uint32_t)f.bin << shift;
        const uint32_t width = (1u << shift) - 1;
        lo = hi - lo > width ? hi - width : lo;
    }
    return goal.end(lo, n, r.by_p ? weight_of(r, logit_of<TYPE>(lo), sh.table) : 0, base_count, base_sum);
}

// The border of a row with the workgroup's bins in place and the table filled; `q`: its key bins.
template <int TYPE>
__device__ __forceinline__ Border row_border(BorderShared& sh, const Row& r, const KeyBins& q, const Work& w, int row) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    Border border{kLowest<TYPE> + 1, 0xffffffffu, 0};  // everything above -inf
    if (r.by_k || r.by_p) {
        const unsigned char* from = w.bins + (size_t)row * w.chunks * kBinBytes;
        // this thread's bins, summed over the chunks; their loads go out together (a chunk behind the last is the last one)
        uint32_t c[4] = {0u, 0u, 0u, 0u};
        unsigned long long s[4] = {0ull, 0ull, 0ull, 0ull};
        if (q.on) {  // bins 4 tid ..
            if (4 * tid < q.all) {
                uint4 cs[kMaxChunks];
                unsigned long long between = 0;
#pragma unroll
                for (int i = 0; i < kMaxChunks; ++i)
                    cs[i] = *reinterpret_cast<const uint4*>(from + (size_t)min(i, w.chunks - 1) * kBinBytes + 16 + 16 * tid);
#pragma unroll
                for (int i = 0; i < kMaxChunks; ++i)
                    if (i < w.chunks) {
                        c[0] += cs[i].x;
                        c[1] += cs[i].y;
                        c[2] += cs[i].z;
                        c[3] += cs[i].w;
                    }
                if (q.np / 4 == tid)
                    for (int i = 0; i < w.chunks; ++i)
                        between += *reinterpret_cast<const unsigned long long*>(from + (size_t)i * kBinBytes);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int b = 4 * tid + i;
                    if (b >= q.all) c[i] = 0;  // what the last 16 bytes hold besides
                    if (r.by_p)
                        s[i] = b == q.np ? between : c[i] ? c[i] * weight_of(r, logit_of<TYPE>(key_of_bin(q, b)), sh.table) : 0;
                }
            }
        } else if (2 * tid < kBins) {  // bins 2 tid, 2 tid + 1
            uint2 cs[kMaxChunks];
            ulonglong2 ss[kMaxChunks];
#pragma unroll
            for (int i = 0; i < kMaxChunks; ++i) {
                const unsigned char* p = from + (size_t)min(i, w.chunks - 1) * kBinBytes;
                cs[i] = r.by_k ? *reinterpret_cast<const uint2*>(p + 8 * kBins + 8 * tid) : make_uint2(0, 0);
                ss[i] = r.by_p ? *reinterpret_cast<const ulonglong2*>(p + 16 * tid) : make_ulonglong2(0, 0);
            }
#pragma unroll
            for (int i = 0; i < kMaxChunks; ++i)
                if (i < w.chunks) {
                    c[0] += cs[i].x;
                    c[1] += cs[i].y;
                    s[0] += ss[i].x;
                    s[1] += ss[i].y;
                }
        }
        auto find = [&](const Goal& goal) {
            const uint32_t c2[2] = {c[0], c[1]};
            const unsigned long long s2[2] = {s[0], s[1]};
            const Bin f = q.on ? border_bin<4>(sh, goal, c, s, 0, 0) : border_bin<2>(sh, goal, c2, s2, 0, 0);
            if (f.bin < 0) return Border{kLowest<TYPE> + 1, 0xffffffffu, 0};  // only when the logits change under the kernel
            uint32_t n = f.count, lo, hi;
            if (q.on) {
                lo = f.bin == q.np ? kLeastNegative + 1 : key_of_bin(q, f.bin);
                hi = f.bin == q.np ? kLeastPositive - 1 : lo;
            } else {
                lo = first_key_of_bins<TYPE>(r, f.bin, lane);
                hi = f.bin ? first_key_of_bins<TYPE>(r, f.bin - 1, lane) - 1 : key_of<TYPE>(r.top);
                // entries are counted for top_k only
                if (!r.by_k && lo == hi) n = (uint32_t)(f.sum / weight_of(r, logit_of<TYPE>(lo), sh.table));
            }
            return border_among<TYPE>(sh, r, goal, lo, hi, n, f.before_count, f.before_sum);
        };
        unsigned long long total = 0;
        if (r.by_k) {
            border = find(Goal{true, (uint32_t)r.top_k, 0});
            total = border.sum;
        }
        __syncthreads();  // the slots of the search
        if (r.by_p) {
            if (!r.by_k) {
                total = wave_total(s[0] + s[1] + s[2] + s[3]);
                if (lane == 0) sh.part_sum[wave] = total;
                __syncthreads();
                total = wave_total(lane < kBorderWaves ? sh.part_sum[lane] : 0ull);
                __syncthreads();
            }
            border = find(Goal{false, 0, share_limit(r, total)});
        }
    }
    if (r.min_p > 0.f) {
        const uint32_t k = first_key_of_min_p<TYPE>(r, lane);
        if (k > border.key) border = Border{k, 0xffffffffu, 0};
    }
    return border;
}

template <int TYPE>
__global__ __launch_bounds__(kBorderThreads) void sample_border_kernel(SampleArgs a, Work w) {
    __shared__ BorderShared sh;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1);
    Row r = row_of<TYPE>(a, row);
    int index;
    if (!load_top<TYPE>(r, w, row, lane, index)) return;  // uniform
    fill_table(sh.table, tid);
    __syncthreads();
    const Border border = row_border<TYPE>(sh, r, key_bins<TYPE>(r), w, row);
    if (tid == 0) w.border[row] = make_uint2(border.key, border.ties);
}

// The weight of an entry above the border's key; `tie`: it has that key.
template <int TYPE>
__device__ __forceinline__ unsigned long long kept_weight(const Row& r, float x, uint32_t border, const double* table, bool& tie) {
    const uint32_t k = key_of<TYPE>(x);
    tie = k == border;
    return k > border ? weight_of(r, x, table) : 0;
}

// The weight of a segment's entries above the border's key and the number of those with it, eight entries a lane.
template <int TYPE>
__device__ __forceinline__ unsigned long long segment_weight(const Row& r, const float (&x)[8], uint32_t border,
                                                             const double* table, uint32_t& ties) {
    unsigned long long sum = 0;
    ties = 0;
    float m = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, x[j]);
    if (!__any(key_of<TYPE>(m) >= border)) return 0;  // nothing of the segment is kept
    bool tie;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        sum += kept_weight<TYPE>(r, x[j], border, table, tie);
        ties += tie;
    }
    ties = wave_total(ties);
    return wave_total(sum);
}

template <int TYPE>
__global__ __launch_bounds__(512) void sample_segments_kernel(SampleArgs a, Work w) {
    const int row = blockIdx.x / w.chunks, chunk = blockIdx.x % w.chunks, tid = threadIdx.x, lane = tid & (kWave - 1);
    Row r = row_of<TYPE>(a, row);
    int index;
    if (!load_top<TYPE>(r, w, row, lane, index)) return;  // uniform
    __shared__ double table[32];
    const uint32_t border = w.border[row].x;
    fill_table(table, tid);
    __syncthreads();
    const int per = w.chunk / kSegment, last = min(w.segments, (chunk + 1) * per);
    for (int s = chunk * per + tid / kWave; s < last; s += 512 / kWave) {
        float x[8];
        load8<TYPE>(r.at, kSegment * s + 8 * lane, r.vocab, r.aligned, x);
        uint32_t ties;
        const unsigned long long sum = segment_weight<TYPE>(r, x, border, table, ties);
        if (lane == 0) {
            w.seg[(size_t)row * w.segments + s] = sum;
            w.tie[(size_t)row * w.segments + s] = ties;
        }
    }
}

__device__ __forceinline__ uint32_t ties_kept(uint32_t ties, uint32_t before, uint32_t count) {
    return ties > before ? min(ties - before, count) : 0u;
}

// The draw in segments first .. first + count - 1 of a row, whose weights s and ties n thread i holds for segment first + i.
// Before them lie `before_sum` and `before_ties`; `total`: of the whole row (0: these segments are the whole row).
struct DrawShared {
    unsigned long long part_sum[kBorderWaves], before_sum, all;
    uint32_t part_count[kBorderWaves], before_ties;
    int found;
};
template <int TYPE>
__device__ __forceinline__ void draw_in(DrawShared& sh, const SampleArgs& a, const Row& r, int row, const double* table, uint2 border,
                                        int first, int count, unsigned long long s, uint32_t n, unsigned long long before_sum,
                                        uint32_t before_ties, unsigned long long total) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    if (tid == 0) {
        sh.found = count - 1;
        sh.before_sum = before_sum;
        sh.before_ties = before_ties;
    }
    const uint32_t before = before_ties + block_prefix<uint32_t>(n, sh.part_count, lane, wave) - n;  // and the table is there
    const unsigned long long border_w = weight_of(r, logit_of<TYPE>(border.x), table);
    const unsigned long long mine = s + ties_kept(border.y, before, n) * border_w;
    const unsigned long long through = before_sum + block_prefix<unsigned long long>(mine, sh.part_sum, lane, wave);
    if (tid == kBorderThreads - 1) sh.all = through;
    __syncthreads();
    const unsigned long long target = target_of(a.uniform[row], total ? total : sh.all);
    if (through > target && through - mine <= target) {
        sh.found = tid;
        sh.before_sum = through - mine;
        sh.before_ties = before;
    }
    __syncthreads();
    if (wave != 0) return;
    const int i0 = kSegment * (first + sh.found) + 8 * lane;
    float x[8];
    load8<TYPE>(r.at, i0, r.vocab, r.aligned, x);
    unsigned long long wj[8], sum = 0;
    bool tie[8];
    uint32_t ties = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        wj[j] = kept_weight<TYPE>(r, x[j], border.x, table, tie[j]);
        ties += tie[j];
    }
    uint32_t rank = sh.before_ties + wave_prefix<uint32_t>(ties) - ties;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (tie[j]) wj[j] = rank++ < border.y ? border_w : 0;
        sum += wj[j];
    }
    unsigned long long cum = sh.before_sum + wave_prefix<unsigned long long>(sum) - sum;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (cum <= target && cum + wj[j] > target) a.out[row] = i0 + j;  // one entry's
        cum += wj[j];
    }
}

template <int TYPE>
__global__ __launch_bounds__(kBorderThreads) void sample_draw_kernel(SampleArgs a, Work w) {
    __shared__ double table[32];
    __shared__ DrawShared sh;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1);
    Row r = row_of<TYPE>(a, row);
    int index;
    if (!load_top<TYPE>(r, w, row, lane, index)) {  // uniform
        if (tid == 0) a.out[row] = index;
        return;
    }
    fill_table(table, tid);
    const size_t at = (size_t)row * w.segments + tid;
    const unsigned long long s = tid < w.segments ? w.seg[at] : 0;
    const uint32_t n = tid < w.segments ? w.tie[at] : 0;
    draw_in<TYPE>(sh, a, r, row, table, w.border[row], 0, w.segments, s, n, 0, 0, 0);
}

// Border and draw of a row of bf16 logits.  The key bins say what each chunk's kept entries weigh, so that only the chunk
// with the drawn entry is read again.  A row without key bins, or with its border between them, is read here as a whole.
struct FinishShared {
    BorderShared border;
    DrawShared draw;
    unsigned long long chunk_sum[kMaxChunks][kBorderWaves];
    uint32_t chunk_ties[kMaxChunks];
};
__global__ __launch_bounds__(kBorderThreads) void sample_finish_kernel(SampleArgs a, Work w) {
    constexpr int TYPE = 0;
    __shared__ FinishShared sh;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    Row r = row_of<TYPE>(a, row);
    int index;
    if (!load_top<TYPE>(r, w, row, lane, index)) {  // uniform
        if (tid == 0) a.out[row] = index;
        return;
    }
    const double* table = sh.border.table;
    fill_table(sh.border.table, tid);
    if (tid < kMaxChunks) sh.chunk_ties[tid] = 0;
    __syncthreads();
    const KeyBins q = key_bins<TYPE>(r);
    const Border border = row_border<TYPE>(sh.border, r, q, w, row);
    int first = 0, last = w.segments;
    unsigned long long before_sum = 0, total = 0;
    uint32_t before_ties = 0;
    if (q.on && (border.key >= kLeastPositive || border.key <= kLeastNegative)) {
        const unsigned char* from = w.bins + (size_t)row * w.chunks * kBinBytes;
        const int edge = bin_of_key(q, border.key);  // behind all bins: nothing is cut off
        const bool some = 4 * kWave * wave <= edge && 4 * kWave * wave < q.all;  // of this wave's bins
        uint4 c[kMaxChunks];
        unsigned long long weight[4] = {0ull, 0ull, 0ull, 0ull};
        const int mine = min(4 * tid, q.all - 1) & ~3;
        if (some) {
#pragma unroll
            for (int i = 0; i < kMaxChunks; ++i)
                c[i] = *reinterpret_cast<const uint4*>(from + (size_t)min(i, w.chunks - 1) * kBinBytes + 16 + 4 * mine);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int b = 4 * tid + i;
                if (b < min(edge, q.all) && b != q.np) weight[i] = weight_of(r, logit_of<TYPE>(key_of_bin(q, b)), table);
            }
        }
#pragma unroll
        for (int i = 0; i < kMaxChunks; ++i)
            if (i < w.chunks) {
                unsigned long long s = 0;
                if (some) {
                    s = c[i].x * weight[0] + c[i].y * weight[1] + c[i].z * weight[2] + c[i].w * weight[3];
                    if (q.np / 4 == tid && edge > q.np) s += *reinterpret_cast<const unsigned long long*>(from + (size_t)i * kBinBytes);
                    s = wave_total(s);
                    if (edge / 4 == tid && edge < q.all)
                        sh.chunk_ties[i] = edge % 4 == 0 ? c[i].x : edge % 4 == 1 ? c[i].y : edge % 4 == 2 ? c[i].z : c[i].w;
                }
                if (lane == 0) sh.chunk_sum[i][wave] = s;
            }
        __syncthreads();
        unsigned long long s = 0;
        uint32_t n = 0;
        if (lane < w.chunks) {
            for (int v = 0; v < kBorderWaves; ++v) s += sh.chunk_sum[lane][v];
            n = sh.chunk_ties[lane];
        }
        const uint32_t before = wave_prefix<uint32_t>(n) - n;
        const unsigned long long kept = s + ties_kept(border.ties, before, n) * weight_of(r, logit_of<TYPE>(border.key), table);
        const unsigned long long through = wave_prefix<unsigned long long>(kept);
        total = lane_value(through, kWave - 1);
        const unsigned long long past = __ballot(through > target_of(a.uniform[row], total));
        const int chunk = past ? __builtin_ctzll(past) : w.chunks - 1;
        before_sum = lane_value(through, chunk) - lane_value(kept, chunk);
        before_ties = lane_value(before, chunk);
        const int per = w.chunk / kSegment;
        first = chunk * per;
        last = min(w.segments, first + per);
    }
    __syncthreads();
    walk<TYPE, 5>(r, kSegment * first + 8 * tid, kSegment * last, 8 * kBorderThreads, [&](int i, const float(&x)[8]) {
        uint32_t ties;
        const unsigned long long sum = segment_weight<TYPE>(r, x, border.key, table, ties);  // a wave's entries are a segment
        if (lane == 0) {
            sh.border.sum[i / kSegment - first] = sum;
            sh.border.count[i / kSegment - first] = ties;
        }
    });
    __syncthreads();
    const unsigned long long s = tid < last - first ? sh.border.sum[tid] : 0;
    const uint32_t n = tid < last - first ? sh.border.count[tid] : 0;
    draw_in<TYPE>(sh.draw, a, r, row, table, make_uint2(border.key, border.ties), first, last - first, s, n, before_sum, before_ties,
                  total);
}

// ---------------------------------------------------------------- short rows: one wave a row
constexpr int kWaveBins = kBins / 4, kWaveBinsPerLane = (kWaveBins + kWave - 1) / kWave;  // 8 an octave

struct WaveBins {
    unsigned long long sum[kWaveBinsPerLane * kWave];
    uint32_t count[kWaveBinsPerLane * kWave];
};

// Other lanes' LDS writes before this point are seen behind it (a wave's LDS accesses are carried out in order).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int TYPE, int E>
__device__ Border wave_border(WaveBins& sh, const Row& r, const float (&x)[E], const unsigned long long (&weight)[E],
                              const Goal& goal, int lane) {
    constexpr int PER = kWaveBinsPerLane;
    uint32_t lo = kLowest<TYPE> + 1, hi = key_of<TYPE>(r.top), base_count = 0;
    unsigned long long base_sum = 0;
    int shift = -1;  // -1: bins linear in log w
    for (;;) {
#pragma unroll
        for (int b = 0; b < PER; ++b) {
            sh.sum[PER * lane + b] = 0;
            sh.count[PER * lane + b] = 0;
        }
        wave_sync();
        auto bin_at = [&](float v) {
            const uint32_t k = key_of<TYPE>(v);
            if (k - lo > hi - lo) return kWaveBins;
            if (shift >= 0) return (int)((hi - k) >> shift);
            return bin_of(parts_of(r, v)) / (kBins / kWaveBins);  // the entries without weight: the last
        };
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int b = bin_at(x[e]);
            if (b >= kWaveBins) continue;
            atomicAdd(&sh.count[b], 1u);
            if (weight[e]) atomicAdd(&sh.sum[b], weight[e]);
        }
        wave_sync();
        uint32_t c[PER], ct = 0;
        unsigned long long s[PER], st = 0;
#pragma unroll
        for (int b = 0; b < PER; ++b) {
            c[b] = sh.count[PER * lane + b];
            s[b] = sh.sum[PER * lane + b];
            ct += c[b];
            st += s[b];
        }
        uint32_t cb = base_count + wave_prefix<uint32_t>(ct) - ct, found_c = 0, found_n = 0;
        unsigned long long sb = base_sum + wave_prefix<unsigned long long>(st) - st, found_s = 0;
        int found = -1;
#pragma unroll
        for (int b = 0; b < PER; ++b) {
            if (c[b] && goal.inside(cb, sb)) {
                found = PER * lane + b;
                found_c = cb;
                found_s = sb;
                found_n = c[b];
            }
            cb += c[b];
            sb += s[b];
        }
        const unsigned long long mask = __ballot(found >= 0);
        if (!mask) return Border{kLowest<TYPE> + 1, 0xffffffffu, 0};  // only when the logits change under the kernel
        const int l = 63 - __builtin_clzll(mask);
        const int bin = __builtin_amdgcn_readlane(found, l);
        base_count = lane_value(found_c, l);
        base_sum = lane_value(found_s, l);
        const uint32_t n = lane_value(found_n, l);
        uint32_t kmin = 0xffffffffu, kmax = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (bin_at(x[e]) == bin) {
                kmin = min(kmin, key_of<TYPE>(x[e]));
                kmax = max(kmax, key_of<TYPE>(x[e]));
            }
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            kmin = min(kmin, (uint32_t)__shfl_xor(kmin, d));
            kmax = max(kmax, (uint32_t)__shfl_xor(kmax, d));
        }
        lo = kmin;
        hi = kmax;
        if (lo >= hi) {
            unsigned long long w = 0;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (key_of<TYPE>(x[e]) == lo) w = weight[e];
            return goal.end(lo, n, wave_largest(w), base_count, base_sum);
        }
        shift = max(0, 32 - __builtin_clz(hi - lo) - 8);
        wave_sync();
    }
}

template <int TYPE, int J>
__global__ __launch_bounds__(256) void sample_wave_kernel(SampleArgs a, int rows) {
    constexpr int E = 8 * J;
    __shared__ double table[32];
    __shared__ WaveBins bins[4];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, row = 4 * blockIdx.x + wave;
    fill_table(table, tid);
    __syncthreads();
    if (row >= rows) return;
    Row r = row_of<TYPE>(a, row);
    float x[E];  // entries 8 (lane + 64 j) ..
    unsigned long long code = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        float v[8];
        const int i = 8 * (lane + kWave * j);
        load8<TYPE>(r.at, i, r.vocab, r.aligned, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[8 * j + e] = v[e];
            if (i + e < r.vocab) code = max(code, top_code<TYPE>(v[e], i + e));
        }
    }
    int index;
    if (!take_top<TYPE>(r, wave_largest(code), index)) {
        if (lane == 0) a.out[row] = index;
        return;
    }
    unsigned long long weight[E];
#pragma unroll
    for (int e = 0; e < E; ++e) weight[e] = weight_of(r, x[e], table);
    Border border{kLowest<TYPE> + 1, 0xffffffffu, 0};
    if (r.by_k) border = wave_border<TYPE, E>(bins[wave], r, x, weight, Goal{true, (uint32_t)r.top_k, 0}, lane);
    if (r.by_p) {
        unsigned long long total = border.sum;
        if (!r.by_k) {
#pragma unroll
            for (int e = 0; e < E; ++e) total += weight[e];
            total = wave_total(total);
        }
        border = wave_border<TYPE, E>(bins[wave], r, x, weight, Goal{false, 0, share_limit(r, total)}, lane);
    }
    if (r.min_p > 0.f) {
        const uint32_t k = first_key_of_min_p<TYPE>(r, lane);
        if (k > border.key) border = Border{k, 0xffffffffu, 0};
    }
    // the kept weights in index order
    uint32_t rank = 0;
    unsigned long long total = 0, through[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        uint32_t ties = 0;
#pragma unroll
        for (int e = 8 * j; e < 8 * j + 8; ++e) ties += key_of<TYPE>(x[e]) == border.key;
        const uint32_t all = wave_prefix<uint32_t>(ties);
        uint32_t mine = rank + all - ties;
        rank += lane_value(all, kWave - 1);
        unsigned long long s = 0;
#pragma unroll
        for (int e = 8 * j; e < 8 * j + 8; ++e) {
            const uint32_t k = key_of<TYPE>(x[e]);
            const bool tie = k == border.key, kept = k > border.key || (tie && mine < border.ties);
            mine += tie;
            weight[e] = kept ? weight[e] : 0;
            s += weight[e];
        }
        through[j] = total + wave_prefix<unsigned long long>(s);
        total = lane_value(through[j], kWave - 1);
        through[j] -= s;
    }
    const unsigned long long target = target_of(a.uniform[row], total);
#pragma unroll
    for (int j = 0; j < J; ++j) {
        unsigned long long cum = through[j];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (cum <= target && cum + weight[8 * j + e] > target) a.out[row] = 8 * (lane + kWave * j) + e;  // one entry's
            cum += weight[8 * j + e];
        }
    }
}

// ---------------------------------------------------------------- launches
// Where a call's parts lie in its workspace, and what it needs in all.
struct SamplePlan {
    int chunks, chunk, segments;
    long long bins, seg, border, tie, bytes;  // offsets; the largest logits lie at 0
};

constexpr int kReaders = 1024;  // workgroups that read rows, about, of at least 8 segments each

void lay_out(SamplePlan& p, long long rows, long long chunks) {  // chunks: of all rows
    p.bins = (8 * chunks + 15) / 16 * 16;  // read 16 bytes at a time
    p.seg = p.bins + chunks * kBinBytes;
    p.border = p.seg + 8 * rows * p.segments;
    p.tie = p.border + 8 * rows;
    p.bytes = (p.tie + 4 * rows * p.segments + 15) / 16 * 16;
}

SamplePlan sample_plan(int rows, int vocab) {
    SamplePlan p{};
    if (vocab <= kSmall) return p;
    p.segments = (vocab + kSegment - 1) / kSegment;
    int chunks = kReaders / rows;
    if (chunks > kMaxChunks) chunks = kMaxChunks;
    if (chunks > p.segments / 8) chunks = p.segments / 8;
    if (chunks < 1) chunks = 1;
    p.chunk = (p.segments + chunks - 1) / chunks * kSegment;
    p.chunks = (vocab + p.chunk - 1) / p.chunk;
    lay_out(p, rows, (long long)rows * p.chunks);
    return p;
}

// No call of up to `rows` rows and `vocab` entries needs more, whatever the workgroups that its rows are shared out over.
long long most_bytes(int rows, int vocab) {
    SamplePlan p{};
    if (vocab <= kSmall) return 0;
    p.segments = (vocab + kSegment - 1) / kSegment;
    long long chunks = (long long)rows * (p.segments / 8 < 1 ? 1 : p.segments / 8 < kMaxChunks ? p.segments / 8 : kMaxChunks);
    const long long most = rows > kReaders ? rows : kReaders;
    lay_out(p, rows, chunks < most ? chunks : most);
    return p.bytes;
}

// More bf16 rows than this are drawn by a workgroup each, fewer by several.  Several / one: 28 / 31 us for one row of 151,936
// with top-p (18 / 29 without), 33.5 / 33.8 for 16, 34.9 / 35.0 for 17, 43.7 / 40.9 for 40, 62 / 53 for 128; 28 / 25 for 40 of 5,000,
// 62 / 58 for 400 of 30,000.  Rows without key bins, which the host cannot tell, lose by it while they are long and few: log-
// probabilities 49.7 / 67.9 for 17, 59.6 / 78.9 for 40 and 84.5 / 96.1 for 128 of 151,936, but 36.4 / 31.5 for 40 of 5,000 and
// 84.7 / 73.3 for 400 of 30,000.
constexpr int kFewRows = 16;

template <int TYPE>
int launch_sample(const SampleArgs& a, int rows, const SamplePlan& p, void* ws, hipStream_t st) {
    if (a.vocab <= kSmall) {
        const dim3 grid((unsigned)((rows + 3) / 4));
        if (a.vocab <= 512)
            hipLaunchKernelGGL((sample_wave_kernel<TYPE, 1>), grid, dim3(256), 0, st, a, rows);
        else if (a.vocab <= 1024)
            hipLaunchKernelGGL((sample_wave_kernel<TYPE, 2>), grid, dim3(256), 0, st, a, rows);
        else
            hipLaunchKernelGGL((sample_wave_kernel<TYPE, 4>), grid, dim3(256), 0, st, a, rows);
        return moss_launch_status();
    }
    unsigned char* at = (unsigned char*)ws;
    const Work w{(unsigned long long*)at, at + p.bins, (unsigned long long*)(at + p.seg), (uint32_t*)(at + p.tie),
                 (uint2*)(at + p.border), p.chunks, p.chunk, p.segments,
                 TYPE == 0 && rows > kFewRows};
    const dim3 many((unsigned)(rows * p.chunks)), one((unsigned)rows);
    hipLaunchKernelGGL(sample_top_kernel<TYPE>, many, dim3(512), 0, st, a, w);
    hipLaunchKernelGGL(sample_bins_kernel<TYPE>, many, dim3(512), 0, st, a, w);
    if (w.finish) {
        hipLaunchKernelGGL(sample_finish_kernel, one, dim3(kBorderThreads), 0, st, a, w);
    } else {
        hipLaunchKernelGGL(sample_border_kernel<TYPE>, one, dim3(kBorderThreads), 0, st, a, w);
        hipLaunchKernelGGL(sample_segments_kernel<TYPE>, many, dim3(512), 0, st, a, w);
        hipLaunchKernelGGL(sample_draw_kernel<TYPE>, one, dim3(kBorderThreads), 0, st, a, w);
    }
    return moss_launch_status();
}

}  // namespace
}  // namespace moss

using namespace moss;

// Enough for any call of up to these sizes: fewer rows are read by more workgroups each.
MOSS_API long long moss_sample_rows_workspace_bytes(int rows, int vocab) {
    if (rows <= 0 || rows > (1 << 21) || vocab <= 0 || vocab > kMaxVocab) return 0;
    return most_bytes(rows, vocab);
}

MOSS_API int moss_sample_rows(const void* logits, int dtype, int rows, long long stride, int vocab, const void* uniform,
                              const void* temperature, float temperature_value, const void* top_k, int top_k_value,
                              const void* top_p, float top_p_value, const void* min_p, float min_p_value, void* out,
                              void* workspace, long long workspace_bytes, void* stream) {
    MOSS_CHECK_ARG(logits && uniform && out && rows > 0 && rows <= (1 << 21) && vocab > 0 && vocab <= kMaxVocab &&
                   stride >= vocab && dtype >= 0 && dtype <= 2);
    MOSS_CHECK_ARG(MOSS_ALIGNED(logits, dtype == 2 ? 4 : 2) && MOSS_ALIGNED(uniform, 4) && MOSS_ALIGNED(temperature, 4) &&
                   MOSS_ALIGNED(top_k, 4) && MOSS_ALIGNED(top_p, 4) && MOSS_ALIGNED(min_p, 4) && MOSS_ALIGNED(out, 8));
    const SamplePlan p = sample_plan(rows, vocab);
    MOSS_CHECK_ARG(p.bytes == 0 || (workspace && MOSS_ALIGNED(workspace, 16) && workspace_bytes >= most_bytes(rows, vocab)));
    const SampleArgs a{logits, stride, vocab, (const float*)uniform, (const float*)temperature, (const int*)top_k,
                       (const float*)top_p, (const float*)min_p, temperature_value, top_p_value, min_p_value, top_k_value,
                       (int64_t*)out};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0) return launch_sample<0>(a, rows, p, workspace, st);
    if (dtype == 1) return launch_sample<1>(a, rows, p, workspace, st);
    return launch_sample<2>(a, rows, p, workspace, st);
}
