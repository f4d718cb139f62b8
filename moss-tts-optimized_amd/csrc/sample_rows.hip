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
// What bounds it: the arithmetic of w in 64 bits for every entry, and, for few rows, the chain of steps.  So a row is
// read by several workgroups, in five launches (largest logit; histogram; border; weight of each segment of 512 entries;
// draw), of which the histogram, or the segments' weights, is the one that forms w for every entry: a row without top-k
// and top-p has no histogram, a row with them few weights in its segments.  w takes one table of 2^(-j / 1024), a
// cubic and one fma that also rounds: 16 operations.  A row of up to 2048 entries is one wave's: it holds them and their weights in
// registers, and needs no barrier.
#include "common.h"

namespace moss {
namespace {

constexpr double kOne = 17592186044416.0;  // 2^44: 2^19 entries sum below 2^63
constexpr int kSteps = 1024;               // steps of z in an octave of w
constexpr int kSpan = 46;                  // octaves: smaller weights are 0
constexpr int kBinShift = 5;               // 32 steps a bin
constexpr int kBins = kSpan * kSteps >> kBinShift;
constexpr int kSegment = 512;              // entries
constexpr int kSmall = 2048;               // entries of a row that one wave takes
constexpr int kMaxVocab = 1 << 19;

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

// Eight logits from index i on, as they are compared: NaN below everything, -0 equal to 0, -inf behind the row's end.
template <int TYPE>
__device__ __forceinline__ void load8(const void* row, int i, int vocab, bool aligned, float (&x)[8]) {
    if (aligned && i + 8 <= vocab) {
        if constexpr (TYPE == 2) {
            const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + i);
            const float4 a = p[0], b = p[1];
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
            const u32x4_t w = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint16_t*>(row) + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t word = w[j];
                x[2 * j] = TYPE == 0 ? bf16_lo(word) : half_value(word & 0xffffu);
                x[2 * j + 1] = TYPE == 0 ? bf16_hi(word) : half_value(word >> 16);
            }
        }
    } else {
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
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = x[j] != x[j] ? -INFINITY : x[j] + 0.0f;
}

// Order-preserving key of a logit.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kLowest = 0x007fffffu;  // the key of -inf

// One row's settings, and its largest logit once it is known.
struct Row {
    const void* at;
    int vocab;
    bool aligned;  // 16-byte loads
    float temperature, top_p, min_p;
    int top_k;
    bool by_k, by_p;
    float top;
    double rate;  // steps of z per unit of a logit: kSteps log2(e) / T
};

template <int TYPE>
__device__ __forceinline__ Row row_of(const SampleArgs& a, int i) {
    Row r;
    r.at = reinterpret_cast<const unsigned char*>(a.logits) + (size_t)i * a.stride * (TYPE == 2 ? 4 : 2);
    r.vocab = a.vocab;
    r.aligned = MOSS_ALIGNED(r.at, 16);
    r.temperature = a.temperature ? a.temperature[i] : a.temperature_v;
    r.top_k = a.top_k ? a.top_k[i] : a.top_k_v;
    r.top_p = a.top_p ? a.top_p[i] : a.top_p_v;
    r.min_p = fminf(a.min_p ? a.min_p[i] : a.min_p_v, 1.f);
    r.by_k = r.top_k > 0 && r.top_k < r.vocab;
    r.by_p = r.top_p < 1.f;
    return r;
}

// The largest logit with its first index, as one number whose maximum is looked for (0: none).
__device__ __forceinline__ unsigned long long top_code(float x, int i) {
    return ((unsigned long long)key_of(x) << 32) | (uint32_t)~i;
}
// Sets the row's largest logit; false when there is nothing to draw (then `index` is the answer).
__device__ __forceinline__ bool take_top(Row& r, unsigned long long code, int& index) {
    const uint32_t k = (uint32_t)(code >> 32);
    r.top = logit_of(k);
    index = k > kLowest ? (int)~(uint32_t)code : -1;
    r.rate = (kSteps * 1.4426950408889634) / (double)r.temperature;
    return k > kLowest && r.temperature > 0.f;
}

// How far a logit lies under the largest one, in steps of w (kSpan octaves or more: no weight).
__device__ __forceinline__ double steps_of(const Row& r, float x) {
    return x == r.top ? 0.0 : ((double)r.top - (double)x) * r.rate;
}
__device__ __forceinline__ int bin_of(const Row& r, float x) {
    const double z = steps_of(r, x);
    return z < (double)(kSpan * kSteps) ? (int)z >> kBinShift : kBins;
}
// w 2^44, to the nearest integer: table[j] = 2^(44 - j / kSteps); the cubic is off by 10^-14.
__device__ __forceinline__ unsigned long long weight_of(const Row& r, float x, const double* table) {
    const double z = steps_of(r, x);
    if (!(z < (double)(kSpan * kSteps))) return 0;
    const int zi = (int)z;
    constexpr double c = -0.6931471805599453 / kSteps;
    const double f = (z - (double)zi) * c;
    const double p = table[zi & (kSteps - 1)] * fma(f, fma(f, fma(f, 1.0 / 6.0, 0.5), 1.0), 1.0);
    const double octave = __hiloint2double((1023 - zi / kSteps) << 20, 0);
    return (unsigned long long)__double_as_longlong(fma(p, octave, 4503599627370496.0)) & 0xfffffffffffffull;
}
__device__ __forceinline__ void fill_table(double* table, int tid, int threads) {
    for (int j = tid; j < kSteps; j += threads) table[j] = exp2((double)-j / kSteps) * kOne;
}

// The smallest key up to the largest logit's that fulfils a condition which the largest one does and, once it holds,
// holds for every larger key.  64 keys a turn; every lane gets the answer.
template <typename Fn>
__device__ __forceinline__ uint32_t first_key(uint32_t top, int lane, Fn holds) {
    uint32_t lo = kLowest, hi = top;  // it fails at lo
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + kWave - 1) / kWave;
        const uint32_t k = min(hi - lo, step * (uint32_t)(lane + 1)) + lo;
        const unsigned long long mask = __ballot(k == hi || holds(logit_of(k)));
        const uint32_t l = (uint32_t)__builtin_ctzll(mask);
        hi = min(hi - lo, step * (l + 1)) + lo;
        lo += l ? min(hi - lo - 1, step * l) : 0;
    }
    return hi;
}
__device__ __forceinline__ uint32_t first_key_of_bins(const Row& r, int bin, int lane) {  // of bins 0 .. bin
    return first_key(key_of(r.top), lane, [&](float x) { return bin_of(r, x) <= bin; });
}
__device__ __forceinline__ uint32_t first_key_of_min_p(const Row& r, int lane) {
    return first_key(key_of(r.top), lane, [&](float x) { return exp2(-steps_of(r, x) / kSteps) >= (double)r.min_p; });
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
// The number that the sums through the kept entries are held against.
__device__ __forceinline__ unsigned long long target_of(float u, unsigned long long total) {
    const double goal = (double)u * (double)total;  // u outside [0, 1) draws the first or the last kept entry
    return goal > 0.0 ? min((unsigned long long)fmin(goal, 9.2e18), total - 1) : 0;
}

template <typename V>
__device__ __forceinline__ V wave_prefix(V v, int lane) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const V o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
template <typename V>
__device__ __forceinline__ V wave_total(V v) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) v += __shfl_xor(v, d);
    return v;
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
    v = wave_prefix(v, lane);
    if (lane == kWave - 1) parts[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; ++w) v += parts[w];
    __syncthreads();
    return v;
}

// ---------------------------------------------------------------- long rows: several workgroups a row
struct Work {
    unsigned long long* top;    // [rows, chunks]
    unsigned long long* sum;    // [rows, chunks, kBins]
    uint32_t* count;            // [rows, chunks, kBins]
    unsigned long long* seg;    // [rows, segments]: weight of the entries above the border's key
    uint32_t* tie;              // [rows, segments]: entries with the border's key
    uint2* border;              // [rows]
    int chunks, chunk, segments;  // chunk: entries, whole segments
};

__device__ __forceinline__ bool load_top(Row& r, const Work& w, int row, int lane, int& index) {
    unsigned long long c = 0;
    for (int i = lane; i < w.chunks; i += kWave) c = max(c, w.top[(size_t)row * w.chunks + i]);
    return take_top(r, wave_largest(c), index);
}

template <int TYPE>
__global__ __launch_bounds__(512) void sample_top_kernel(SampleArgs a, Work w) {
    __shared__ unsigned long long parts[8];
    const int row = blockIdx.x / w.chunks, chunk = blockIdx.x % w.chunks, tid = threadIdx.x, lane = tid & (kWave - 1);
    const Row r = row_of<TYPE>(a, row);
    const int end = min(r.vocab, (chunk + 1) * w.chunk);
    unsigned long long best = 0;
    for (int i = chunk * w.chunk + 8 * tid; i < end; i += 8 * 512) {
        float x[8];
        load8<TYPE>(r.at, i, r.vocab, r.aligned, x);
        float m = x[0];
        int at = 0;
#pragma unroll
        for (int j = 1; j < 8; ++j)
            if (x[j] > m) m = x[j], at = j;
        best = max(best, top_code(m, i + at));
    }
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
    __shared__ double table[kSteps];
    __shared__ unsigned long long sum[kBins];
    __shared__ uint32_t count[kBins];
    const int row = blockIdx.x / w.chunks, chunk = blockIdx.x % w.chunks, tid = threadIdx.x, lane = tid & (kWave - 1);
    Row r = row_of<TYPE>(a, row);
    int index;
    if (!(r.by_k || r.by_p) || !load_top(r, w, row, lane, index)) return;  // uniform
    if (r.by_p) fill_table(table, tid, 512);
    for (int b = tid; b < kBins; b += 512) {
        sum[b] = 0;
        count[b] = 0;
    }
    __syncthreads();
    const int end = min(r.vocab, (chunk + 1) * w.chunk);
    for (int i = chunk * w.chunk + 8 * tid; i < end; i += 8 * 512) {
        float x[8];
        load8<TYPE>(r.at, i, r.vocab, r.aligned, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int b = bin_of(r, x[j]);
            if (b >= kBins) continue;
            atomicAdd(&count[b], 1u);
            if (r.by_p) atomicAdd(&sum[b], weight_of(r, x[j], table));
        }
    }
    __syncthreads();
    const size_t at = ((size_t)row * w.chunks + chunk) * kBins;
    for (int b = tid; b < kBins; b += 512) {
        w.count[at + b] = count[b];
        w.sum[at + b] = sum[b];
    }
}

constexpr int kBorderThreads = 1024, kBorderWaves = kBorderThreads / kWave;
constexpr int kList = 2048;

struct BorderShared {
    double table[kSteps];
    unsigned long long sum[2048];
    uint32_t count[2048];
    unsigned long long list_w[kList];
    uint32_t list[kList];
    unsigned long long part_sum[kBorderWaves];
    uint32_t part_count[kBorderWaves], part_min[kBorderWaves], part_max[kBorderWaves];
    unsigned long long before_sum;
    uint32_t before_count, listed, lowest, equal;
    int found;
};

// The last of the 2048 bins in sh whose first entry is inside, given what lies above them; -1: none.  Leaves what lies
// above that bin in sh.before_*.
__device__ __forceinline__ int border_bin(BorderShared& sh, const Goal& goal, uint32_t base_count, unsigned long long base_sum) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const uint32_t c0 = sh.count[2 * tid], c1 = sh.count[2 * tid + 1];
    const unsigned long long s0 = sh.sum[2 * tid], s1 = sh.sum[2 * tid + 1];
    if (tid == 0) sh.found = -1;
    const uint32_t cb = base_count + block_prefix<uint32_t>(c0 + c1, sh.part_count, lane, wave) - c0 - c1;
    const unsigned long long sb = base_sum + block_prefix<unsigned long long>(s0 + s1, sh.part_sum, lane, wave) - s0 - s1;
    if (c1 && goal.inside(cb + c0, sb + s0))
        atomicMax(&sh.found, 2 * tid + 1);
    else if (c0 && goal.inside(cb, sb))
        atomicMax(&sh.found, 2 * tid);
    __syncthreads();
    const int bin = sh.found;
    if (bin >= 0 && bin / 2 == tid) {
        sh.before_count = bin & 1 ? cb + c0 : cb;
        sh.before_sum = bin & 1 ? sb + s0 : sb;
    }
    __syncthreads();
    return bin;
}

// The border inside the keys lo .. hi, which n entries have, behind the given ones.  (Entries that an earlier border left
// out weigh on no decision: what lies before them already exceeds the limit.)
template <int TYPE>
__device__ Border border_among(BorderShared& sh, const Row& r, const Goal& goal, uint32_t lo, uint32_t hi, uint32_t n,
                               uint32_t base_count, unsigned long long base_sum) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    if (n <= kList) {
        // few: collect them; an entry knows what lies above it by looking at all of them
        if (tid == 0) sh.listed = 0;
        if (tid == 0) sh.lowest = 0xffffffffu;
        if (tid == 0) sh.equal = 0;
        __syncthreads();
        for (int i = 8 * tid; i < r.vocab; i += 8 * kBorderThreads) {
            float x[8];
            load8<TYPE>(r.at, i, r.vocab, r.aligned, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t k = key_of(x[j]);
                if (k - lo > hi - lo) continue;
                const uint32_t at = atomicAdd(&sh.listed, 1u);
                if (at >= kList) continue;
                sh.list[at] = k;
                sh.list_w[at] = r.by_p ? weight_of(r, x[j], sh.table) : 0;
            }
        }
        __syncthreads();
        const uint32_t m = min(sh.listed, (uint32_t)kList);
        for (uint32_t e = tid; e < m; e += kBorderThreads) {
            const uint32_t k = sh.list[e];
            uint32_t c = base_count;
            unsigned long long s = base_sum;
            for (uint32_t o = 0; o < m; ++o)
                if (sh.list[o] > k) {
                    ++c;
                    s += sh.list_w[o];
                }
            if (goal.inside(c, s)) atomicMin(&sh.lowest, k);
        }
        __syncthreads();
        const uint32_t key = sh.lowest;
        for (uint32_t e = tid; e < m; e += kBorderThreads) {
            if (sh.list[e] == key) atomicAdd(&sh.equal, 1u);
        }
        // what lies above the border's key
        uint32_t c = 0;
        unsigned long long s = 0;
        for (uint32_t e = tid; e < m; e += kBorderThreads)
            if (sh.list[e] > key) {
                ++c;
                s += sh.list_w[e];
            }
        c = wave_total(c);
        s = wave_total(s);
        if (lane == 0) {
            sh.part_count[wave] = c;
            sh.part_sum[wave] = s;
        }
        __syncthreads();
        c = base_count;
        s = base_sum;
        for (int v = 0; v < kBorderWaves; ++v) {
            c += sh.part_count[v];
            s += sh.part_sum[v];
        }
        const uint32_t equal = sh.equal;
        __syncthreads();
        if (equal == 0) return Border{kLowest + 1, 0xffffffffu, 0};  // only when the logits change under the kernel
        return goal.end(key, equal, !r.by_p ? 0 : weight_of(r, logit_of(key), sh.table), c, s);
    }
    // many: bins over equal parts of the keys' range, until a bin is one key
    while (lo != hi) {
        const uint32_t range = hi - lo;
        const int shift = max(0, 32 - __builtin_clz(range) - 11);
        for (int b = tid; b < 2048; b += kBorderThreads) {
            sh.sum[b] = 0;
            sh.count[b] = 0;
        }
        __syncthreads();
        for (int i = 8 * tid; i < r.vocab; i += 8 * kBorderThreads) {
            float x[8];
            load8<TYPE>(r.at, i, r.vocab, r.aligned, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t k = key_of(x[j]);
                if (k - lo > range) continue;
                atomicAdd(&sh.count[(hi - k) >> shift], 1u);
                if (r.by_p) atomicAdd(&sh.sum[(hi - k) >> shift], weight_of(r, x[j], sh.table));
            }
        }
        __syncthreads();
        const int bin = border_bin(sh, goal, base_count, base_sum);
        if (bin < 0) return Border{kLowest + 1, 0xffffffffu, 0};  // only when the logits change under the kernel
        base_count = sh.before_count;
        base_sum = sh.before_sum;
        n = sh.count[bin];
        hi -= (uint32_t)bin << shift;
        lo = max(lo, hi - ((1u << shift) - 1));  // keys of numbers lie above 2^22, so this does not wrap
        __syncthreads();
        if (shift == 0) break;
    }
    lo = hi;
    return goal.end(lo, n, !r.by_p ? 0 : weight_of(r, logit_of(lo), sh.table), base_count, base_sum);
}

template <int TYPE>
__global__ __launch_bounds__(kBorderThreads) void sample_border_kernel(SampleArgs a, Work w) {
    __shared__ BorderShared sh;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    Row r = row_of<TYPE>(a, row);
    int index;
    if (!load_top(r, w, row, lane, index)) return;  // uniform
    Border border{kLowest + 1, 0xffffffffu, 0};     // everything above -inf
    unsigned long long total = 0;
    auto load_bins = [&]() {
        unsigned long long all = 0;
        for (int b = tid; b < 2048; b += kBorderThreads) {
            uint32_t c = 0;
            unsigned long long s = 0;
            if (b < kBins)
                for (int i = 0; i < w.chunks; ++i) {
                    const size_t at = ((size_t)row * w.chunks + i) * kBins + b;
                    c += w.count[at];
                    s += w.sum[at];
                }
            sh.count[b] = c;
            sh.sum[b] = s;
            all += s;
        }
        __syncthreads();
        return all;
    };
    auto find = [&](const Goal& goal) {
        const int bin = border_bin(sh, goal, 0, 0);
        if (bin < 0) return Border{kLowest + 1, 0xffffffffu, 0};  // only when the logits change under the kernel
        const uint32_t n = sh.count[bin], count = sh.before_count;
        const unsigned long long sum = sh.before_sum;
        const uint32_t lo = first_key_of_bins(r, bin, lane);
        const uint32_t hi = bin ? first_key_of_bins(r, bin - 1, lane) - 1 : key_of(r.top);
        __syncthreads();
        return border_among<TYPE>(sh, r, goal, lo, hi, n, count, sum);
    };
    if (r.by_k || r.by_p) {
        if (r.by_p) fill_table(sh.table, tid, kBorderThreads);
        total = load_bins();
        if (r.by_k) {
            border = find(Goal{true, (uint32_t)r.top_k, 0});
            total = border.sum;
            if (r.by_p) {
                __syncthreads();
                load_bins();
            }
        } else {
            total = wave_total(total);
            if (lane == 0) sh.part_sum[wave] = total;
            __syncthreads();
            total = 0;
            for (int v = 0; v < kBorderWaves; ++v) total += sh.part_sum[v];
            __syncthreads();
        }
        if (r.by_p) border = find(Goal{false, 0, share_limit(r, total)});
    }
    if (r.min_p > 0.f) {
        const uint32_t k = first_key_of_min_p(r, lane);
        if (k > border.key) border = Border{k, 0xffffffffu, 0};
    }
    if (tid == 0) w.border[row] = make_uint2(border.key, border.ties);
}

// The weight of an entry above the border's key; `tie`: it has that key.
__device__ __forceinline__ unsigned long long kept_weight(const Row& r, float x, uint32_t border, const double* table, bool& tie) {
    const uint32_t k = key_of(x);
    tie = k == border;
    return k > border ? weight_of(r, x, table) : 0;
}

template <int TYPE>
__global__ __launch_bounds__(512) void sample_segments_kernel(SampleArgs a, Work w) {
    __shared__ double table[kSteps];
    const int row = blockIdx.x / w.chunks, chunk = blockIdx.x % w.chunks, tid = threadIdx.x, lane = tid & (kWave - 1);
    Row r = row_of<TYPE>(a, row);
    int index;
    if (!load_top(r, w, row, lane, index)) return;  // uniform
    const uint32_t border = w.border[row].x;
    fill_table(table, tid, 512);
    __syncthreads();
    const int per = w.chunk / kSegment, last = min(w.segments, (chunk + 1) * per);
    for (int s = chunk * per + tid / kWave; s < last; s += 512 / kWave) {
        float x[8];
        load8<TYPE>(r.at, kSegment * s + 8 * lane, r.vocab, r.aligned, x);
        unsigned long long sum = 0;
        uint32_t ties = 0;
        float m = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) m = fmaxf(m, x[j]);
        if (__any(key_of(m) >= border)) {  // else nothing of the segment is kept
            bool tie;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum += kept_weight(r, x[j], border, table, tie);
                ties += tie;
            }
            sum = wave_total(sum);
            ties = wave_total(ties);
        }
        if (lane == 0) {
            w.seg[(size_t)row * w.segments + s] = sum;
            w.tie[(size_t)row * w.segments + s] = ties;
        }
    }
}

__device__ __forceinline__ uint32_t ties_kept(uint32_t ties, uint32_t before, uint32_t count) {
    return ties > before ? min(ties - before, count) : 0u;
}

template <int TYPE>
__global__ __launch_bounds__(1024) void sample_draw_kernel(SampleArgs a, Work w) {
    __shared__ double table[kSteps];
    __shared__ unsigned long long part_sum[16], before_sum, all;
    __shared__ uint32_t part_count[16], before_ties;
    __shared__ int found;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    Row r = row_of<TYPE>(a, row);
    int index;
    if (!load_top(r, w, row, lane, index)) {  // uniform
        if (tid == 0) a.out[row] = index;
        return;
    }
    const uint2 border = w.border[row];
    fill_table(table, tid, 1024);
    const size_t at = (size_t)row * w.segments + tid;
    const unsigned long long s = tid < w.segments ? w.seg[at] : 0;
    const uint32_t n = tid < w.segments ? w.tie[at] : 0;
    if (tid == 0) {
        found = w.segments - 1;
        before_sum = 0;
        before_ties = 0;
    }
    const uint32_t before = block_prefix<uint32_t>(n, part_count, lane, wave) - n;  // also the table's barrier
    const unsigned long long border_w = weight_of(r, logit_of(border.x), table);
    const unsigned long long mine = s + ties_kept(border.y, before, n) * border_w;
    const unsigned long long through = block_prefix<unsigned long long>(mine, part_sum, lane, wave);
    if (tid == 1023) all = through;
    __syncthreads();
    const unsigned long long target = target_of(a.uniform[row], all);
    if (through > target && through - mine <= target) {
        found = tid;
        before_sum = through - mine;
        before_ties = before;
    }
    __syncthreads();
    if (wave != 0) return;
    const int i0 = kSegment * found + 8 * lane;
    float x[8];
    load8<TYPE>(r.at, i0, r.vocab, r.aligned, x);
    unsigned long long wj[8], sum = 0;
    bool tie[8];
    uint32_t ties = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        wj[j] = kept_weight(r, x[j], border.x, table, tie[j]);
        ties += tie[j];
    }
    uint32_t rank = before_ties + wave_prefix<uint32_t>(ties, lane) - ties;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (tie[j]) wj[j] = rank++ < border.y ? border_w : 0;
        sum += wj[j];
    }
    unsigned long long cum = before_sum + wave_prefix<unsigned long long>(sum, lane) - sum;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (cum <= target && cum + wj[j] > target) a.out[row] = i0 + j;  // one entry's
        cum += wj[j];
    }
}

// ---------------------------------------------------------------- short rows: one wave a row
constexpr int kWaveBinShift = 7, kWaveBins = 384;  // 46 octaves of 8 bins, 6 bins a lane
static_assert((kSpan * kSteps >> kWaveBinShift) <= kWaveBins && kWaveBins % kWave == 0, "bins");

struct WaveBins {
    unsigned long long sum[kWaveBins];
    uint32_t count[kWaveBins];
};

// Other lanes' LDS writes before this point are seen behind it (a wave's LDS accesses are carried out in order).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int E>
__device__ Border wave_border(WaveBins& sh, const Row& r, const float (&x)[E], const unsigned long long (&weight)[E],
                              const Goal& goal, int lane) {
    constexpr int PER = kWaveBins / kWave;
    uint32_t lo = kLowest + 1, hi = key_of(r.top), base_count = 0;
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
            const uint32_t k = key_of(v);
            if (k - lo > hi - lo) return kWaveBins;
            if (shift >= 0) return (int)((hi - k) >> shift);
            const int b = bin_of(r, v);
            return b >= kBins ? kWaveBins : b >> (kWaveBinShift - kBinShift);
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
        uint32_t cb = base_count + wave_prefix<uint32_t>(ct, lane) - ct, found_c = 0, found_n = 0;
        unsigned long long sb = base_sum + wave_prefix<unsigned long long>(st, lane) - st, found_s = 0;
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
        if (!mask) return Border{kLowest + 1, 0xffffffffu, 0};  // only when the logits change under the kernel
        const int l = 63 - __builtin_clzll(mask);
        const int bin = __shfl(found, l);
        base_count = __shfl(found_c, l);
        base_sum = __shfl(found_s, l);
        const uint32_t n = __shfl(found_n, l);
        uint32_t kmin = 0xffffffffu, kmax = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (bin_at(x[e]) == bin) {
                kmin = min(kmin, key_of(x[e]));
                kmax = max(kmax, key_of(x[e]));
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
                if (key_of(x[e]) == lo) w = weight[e];
            return goal.end(lo, n, wave_largest(w), base_count, base_sum);
        }
        shift = max(0, 32 - __builtin_clz(hi - lo) - 8);
        wave_sync();
    }
}

template <int TYPE, int J>
__global__ __launch_bounds__(256) void sample_wave_kernel(SampleArgs a, int rows) {
    constexpr int E = 8 * J;
    __shared__ double table[kSteps];
    __shared__ WaveBins bins[4];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, row = 4 * blockIdx.x + wave;
    fill_table(table, tid, 256);
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
            if (i + e < r.vocab) code = max(code, top_code(v[e], i + e));
        }
    }
    int index;
    if (!take_top(r, wave_largest(code), index)) {
        if (lane == 0) a.out[row] = index;
        return;
    }
    unsigned long long weight[E];
#pragma unroll
    for (int e = 0; e < E; ++e) weight[e] = weight_of(r, x[e], table);
    Border border{kLowest + 1, 0xffffffffu, 0};
    if (r.by_k) border = wave_border<E>(bins[wave], r, x, weight, Goal{true, (uint32_t)r.top_k, 0}, lane);
    if (r.by_p) {
        unsigned long long total = border.sum;
        if (!r.by_k) {
#pragma unroll
            for (int e = 0; e < E; ++e) total += weight[e];
            total = wave_total(total);
        }
        border = wave_border<E>(bins[wave], r, x, weight, Goal{false, 0, share_limit(r, total)}, lane);
    }
    if (r.min_p > 0.f) {
        const uint32_t k = first_key_of_min_p(r, lane);
        if (k > border.key) border = Border{k, 0xffffffffu, 0};
    }
    // the kept weights in index order
    uint32_t rank = 0;
    unsigned long long total = 0, through[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        uint32_t ties = 0;
#pragma unroll
        for (int e = 8 * j; e < 8 * j + 8; ++e) ties += key_of(x[e]) == border.key;
        const uint32_t all = wave_prefix<uint32_t>(ties, lane);
        uint32_t mine = rank + all - ties;
        rank += __shfl(all, kWave - 1);
        unsigned long long s = 0;
#pragma unroll
        for (int e = 8 * j; e < 8 * j + 8; ++e) {
            const uint32_t k = key_of(x[e]);
            const bool tie = k == border.key, kept = k > border.key || (tie && mine < border.ties);
            mine += tie;
            weight[e] = kept ? weight[e] : 0;
            s += weight[e];
        }
        through[j] = total + wave_prefix<unsigned long long>(s, lane);
        total = __shfl(through[j], kWave - 1);
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
struct SamplePlan {
    int chunks, chunk, segments;
    long long top, sum, seg, border, count, tie, bytes;  // offsets
};

SamplePlan sample_plan(int rows, int vocab) {
    SamplePlan p{};
    if (vocab <= kSmall) return p;
    p.segments = (vocab + kSegment - 1) / kSegment;
    // about 1024 workgroups, of at least 8 segments each and at most 16 a row
    int chunks = 1024 / rows;
    if (chunks > 16) chunks = 16;
    if (chunks > p.segments / 8) chunks = p.segments / 8;
    if (chunks < 1) chunks = 1;
    p.chunk = (p.segments + chunks - 1) / chunks * kSegment;
    p.chunks = (vocab + p.chunk - 1) / p.chunk;
    const long long bins = (long long)rows * p.chunks * kBins, segs = (long long)rows * p.segments;
    p.top = 0;
    p.sum = p.top + 8ll * rows * p.chunks;
    p.seg = p.sum + 8 * bins;
    p.border = p.seg + 8 * segs;
    p.count = p.border + 8ll * rows;
    p.tie = p.count + 4 * bins;
    p.bytes = (p.tie + 4 * segs + 15) / 16 * 16;
    return p;
}

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
    const Work w{(unsigned long long*)(at + p.top), (unsigned long long*)(at + p.sum), (uint32_t*)(at + p.count),
                 (unsigned long long*)(at + p.seg), (uint32_t*)(at + p.tie),           (uint2*)(at + p.border),
                 p.chunks,                          p.chunk,                           p.segments};
    const dim3 many((unsigned)(rows * p.chunks)), one((unsigned)rows);
    hipLaunchKernelGGL(sample_top_kernel<TYPE>, many, dim3(512), 0, st, a, w);
    hipLaunchKernelGGL(sample_bins_kernel<TYPE>, many, dim3(512), 0, st, a, w);
    hipLaunchKernelGGL(sample_border_kernel<TYPE>, one, dim3(kBorderThreads), 0, st, a, w);
    hipLaunchKernelGGL(sample_segments_kernel<TYPE>, many, dim3(512), 0, st, a, w);
    hipLaunchKernelGGL(sample_draw_kernel<TYPE>, one, dim3(1024), 0, st, a, w);
    return moss_launch_status();
}

}  // namespace
}  // namespace moss

using namespace moss;

MOSS_API long long moss_sample_rows_workspace_bytes(int rows, int vocab) {
    if (rows <= 0 || rows > (1 << 21) || vocab <= 0 || vocab > kMaxVocab) return 0;
    return sample_plan(rows, vocab).bytes;
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
    MOSS_CHECK_ARG(p.bytes == 0 || (workspace && MOSS_ALIGNED(workspace, 16) && workspace_bytes >= p.bytes));
    const SampleArgs a{logits, stride, vocab, (const float*)uniform, (const float*)temperature, (const int*)top_k,
                       (const float*)top_p, (const float*)min_p, temperature_value, top_p_value, min_p_value, top_k_value,
                       (int64_t*)out};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0) return launch_sample<0>(a, rows, p, workspace, st);
    if (dtype == 1) return launch_sample<1>(a, rows, p, workspace, st);
    return launch_sample<2>(a, rows, p, workspace, st);
}
