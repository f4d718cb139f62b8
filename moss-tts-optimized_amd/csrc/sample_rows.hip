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
// The borders of the prefix are found without sorting: a histogram (count and sum of w) over 2048 bins that are linear
// in log w, then over 2048 equal parts of the border bin's range of sort keys, until a bin is one key; of the entries
// with that key, the first few in index order are kept.
#include "common.h"

namespace moss {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kBins = 2048;
constexpr double kOne = 17592186044416.0;  // 2^44: vocab up to 2^19 entries sum below 2^63
constexpr double kSpan = 46.0;             // log2 of the smallest weight that is not 0, rounded up

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

struct Row {
    float top;    // the largest logit
    double rate;  // log2(e) / T
    const void* at;
    int vocab;
    bool aligned;  // 16-byte loads
};

__device__ __forceinline__ double share_of(const Row& r, float x) {
    return x == r.top ? 1.0 : exp2(((double)x - (double)r.top) * r.rate);
}
__device__ __forceinline__ unsigned long long weight_of(const Row& r, float x) {
    return (unsigned long long)rint(share_of(r, x) * kOne);
}

// The row's entries, eight at a time: fn(index, x).
template <int TYPE, typename Fn>
__device__ __forceinline__ void each(const Row& r, Fn fn) {
    for (int i = 8 * (int)threadIdx.x; i < r.vocab; i += 8 * kThreads) {
        float x[8];
        load8<TYPE>(r.at, i, r.vocab, r.aligned, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) fn(i + j, x[j]);
    }
}

// Bin of a logit: falls from the largest one on; kBins: no weight.
__device__ __forceinline__ int bin_of(const Row& r, float x) {
    const double y = ((double)r.top - (double)x) * r.rate * (kBins / kSpan);
    return x == r.top ? 0 : y < (double)kBins ? (int)y : kBins;
}

struct Shared {
    unsigned long long sum[kBins];  // later the weights of the segments
    uint32_t count[kBins];          // later their ties
    unsigned long long part_sum[kWaves];
    uint32_t part_count[kWaves], part_min[kWaves], part_max[kWaves];
    int found;
    uint32_t before_count;
    unsigned long long before_sum;
};

// The border of the prefix: entries with a key above `key` are inside, and the first `ties` with that key.
struct Border {
    uint32_t key;
    uint32_t ties;
    unsigned long long sum;  // of the entries inside
};

// Finds the last entry inside: the first `need` entries (by_count), or the entries whose predecessors' sum is at most
// `limit`.  Entries beyond `within` do not exist.
template <int TYPE>
__device__ Border find_border(Shared& sh, const Row& r, bool by_count, uint32_t need, unsigned long long limit,
                              Border within) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    uint32_t base_count = 0;  // entries and weight above the bins looked at
    unsigned long long base_sum = 0;
    uint32_t lo = 0, hi = 0xffffffffu;
    int shift = -1;  // -1: the bins that are linear in log w; else (hi - key) >> shift
    for (;;) {
        for (int i = tid; i < kBins; i += kThreads) {
            sh.count[i] = 0;
            sh.sum[i] = 0;
        }
        __syncthreads();
        each<TYPE>(r, [&](int, float x) {
            const uint32_t k = key_of(x);
            if (k < within.key || k < lo || k > hi) return;
            const int bin = shift < 0 ? bin_of(r, x) : (int)((hi - k) >> shift);
            if (bin >= kBins) return;
            atomicAdd(&sh.count[bin], 1u);
            atomicAdd(&sh.sum[bin], weight_of(r, x));
        });
        __syncthreads();
        // the bin with the border: the last one whose predecessors leave its first entry inside
        uint32_t c0 = sh.count[2 * tid], c1 = sh.count[2 * tid + 1];
        unsigned long long s0 = sh.sum[2 * tid], s1 = sh.sum[2 * tid + 1];
        uint32_t ci = c0 + c1;
        unsigned long long si = s0 + s1;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const uint32_t c = __shfl_up(ci, d);
            const unsigned long long s = __shfl_up(si, d);
            if (lane >= d) {
                ci += c;
                si += s;
            }
        }
        if (lane == kWave - 1) {
            sh.part_count[wave] = ci;
            sh.part_sum[wave] = si;
        }
        if (tid == 0) sh.found = -1;
        __syncthreads();
        uint32_t cb = base_count + ci - c0 - c1;
        unsigned long long sb = base_sum + si - s0 - s1;
        for (int v = 0; v < wave; ++v) {
            cb += sh.part_count[v];
            sb += sh.part_sum[v];
        }
        auto inside = [&](uint32_t c, unsigned long long s) { return by_count ? c < need : s <= limit; };
        const bool in0 = c0 && inside(cb, sb), in1 = c1 && inside(cb + c0, sb + s0);
        if (in1)
            atomicMax(&sh.found, 2 * tid + 1);
        else if (in0)
            atomicMax(&sh.found, 2 * tid);
        __syncthreads();
        const int bin = sh.found;  // the first bin that holds anything is inside, so there is one
        if (bin < 0) return within;  // unless the logits change under the kernel: end all the same
        if (bin == 2 * tid || bin == 2 * tid + 1) {
            sh.before_count = bin & 1 ? cb + c0 : cb;
            sh.before_sum = bin & 1 ? sb + s0 : sb;
        }
        // its range of keys
        uint32_t kmin = 0xffffffffu, kmax = 0;
        each<TYPE>(r, [&](int, float x) {
            const uint32_t k = key_of(x);
            if (k < within.key || k < lo || k > hi) return;
            if ((shift < 0 ? bin_of(r, x) : (int)((hi - k) >> shift)) != bin) return;
            kmin = min(kmin, k);
            kmax = max(kmax, k);
        });
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            kmin = min(kmin, (uint32_t)__shfl_xor(kmin, d));
            kmax = max(kmax, (uint32_t)__shfl_xor(kmax, d));
        }
        if (lane == 0) {
            sh.part_min[wave] = kmin;
            sh.part_max[wave] = kmax;
        }
        __syncthreads();
        base_count = sh.before_count;
        base_sum = sh.before_sum;
        uint32_t n = sh.count[bin];
        lo = 0xffffffffu;
        hi = 0;
        for (int v = 0; v < kWaves; ++v) {
            lo = min(lo, sh.part_min[v]);
            hi = max(hi, sh.part_max[v]);
        }
        __syncthreads();  // the bins are read before they are cleared
        if (lo == hi) {
            // one key: its entries weigh the same
            const unsigned long long w = weight_of(r, logit_of(lo));
            if (lo == within.key) n = min(n, within.ties);
            uint32_t ties = n;
            if (by_count)
                ties = min(n, need - base_count);
            else if (w)
                ties = (uint32_t)min((unsigned long long)n, (limit - base_sum) / w + 1);
            return Border{lo, ties, base_sum + ties * w};
        }
        const uint32_t range = hi - lo;
        shift = max(0, 32 - __builtin_clz(range) - 11);
    }
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

template <int TYPE>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, rowi = blockIdx.x;
    Row r;
    r.at = reinterpret_cast<const unsigned char*>(a.logits) + (size_t)rowi * a.stride * (TYPE == 2 ? 4 : 2);
    r.vocab = a.vocab;
    r.aligned = MOSS_ALIGNED(r.at, 16);
    const float temperature = a.temperature ? a.temperature[rowi] : a.temperature_v;
    const int top_k = a.top_k ? a.top_k[rowi] : a.top_k_v;
    const float top_p = a.top_p ? a.top_p[rowi] : a.top_p_v;
    const float min_p = fminf(a.min_p ? a.min_p[rowi] : a.min_p_v, 1.f);

    // the largest logit and its first index
    uint32_t best = 0;
    int at = 0x7fffffff;
    each<TYPE>(r, [&](int i, float x) {
        const uint32_t k = key_of(x);
        if (k > best) {
            best = k;
            at = i;
        }
    });
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const uint32_t k = __shfl_xor(best, d);
        const int i = __shfl_xor(at, d);
        if (k > best || (k == best && i < at)) {
            best = k;
            at = i;
        }
    }
    if (lane == 0) {
        sh.part_max[wave] = best;
        sh.part_count[wave] = (uint32_t)at;
    }
    __syncthreads();
    for (int v = 0; v < kWaves; ++v) {
        const uint32_t k = sh.part_max[v];
        const int i = (int)sh.part_count[v];
        if (k > best || (k == best && i < at)) {
            best = k;
            at = i;
        }
    }
    __syncthreads();
    r.top = logit_of(best);
    if (r.top == -INFINITY || !(temperature > 0.f)) {
        if (tid == 0) a.out[rowi] = r.top == -INFINITY ? -1 : at;
        return;
    }
    r.rate = 1.4426950408889634 / (double)temperature;

    const bool by_k = top_k > 0 && top_k < r.vocab;
    Border border{key_of(-INFINITY) + 1, 0xffffffffu, 0};  // everything above -inf
    if (by_k) border = find_border<TYPE>(sh, r, true, (uint32_t)top_k, 0, border);
    if (top_p < 1.f) {
        unsigned long long total = border.sum;
        if (!by_k) {
            each<TYPE>(r, [&](int, float x) { total += weight_of(r, x); });
#pragma unroll
            for (int d = 1; d < kWave; d <<= 1) total += __shfl_xor(total, d);
            if (lane == 0) sh.part_sum[wave] = total;
            __syncthreads();
            total = 0;
            for (int v = 0; v < kWaves; ++v) total += sh.part_sum[v];
            __syncthreads();
        }
        border = find_border<TYPE>(sh, r, false, 0, (unsigned long long)((double)fmaxf(top_p, 0.f) * (double)total), border);
    }
    const float border_x = logit_of(border.key);
    const bool border_heavy = !(share_of(r, border_x) < (double)min_p);
    const unsigned long long border_w = border_heavy ? weight_of(r, border_x) : 0;

    // a segment is what a wave reads at once, 512 entries: the weight above the border's key, and the entries on it
    const int segments = (r.vocab + 8 * kWave - 1) / (8 * kWave);
    auto weigh = [&](float x, unsigned long long& w, bool& tie) {
        const uint32_t k = key_of(x);
        tie = k == border.key;
        w = 0;
        if (k <= border.key) return;
        const double share = share_of(r, x);
        if (!(share < (double)min_p)) w = (unsigned long long)rint(share * kOne);
    };
    for (int s = wave; s < segments; s += kWaves) {
        float x[8];
        load8<TYPE>(r.at, 8 * (kWave * s + lane), r.vocab, r.aligned, x);
        unsigned long long w = 0, wj;
        uint32_t n = 0;
        bool tie;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            weigh(x[j], wj, tie);
            w += wj;
            n += tie;
        }
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            w += __shfl_xor(w, d);
            n += __shfl_xor(n, d);
        }
        if (lane == 0) {
            sh.sum[s] = w;
            sh.count[s] = n;
        }
    }
    if (tid == 0) sh.found = segments - 1;
    __syncthreads();
    const uint32_t n = tid < segments ? sh.count[tid] : 0;
    const uint32_t ties_before = block_prefix<uint32_t>(n, sh.part_count, lane, wave) - n;
    auto ties_kept = [&](uint32_t before, uint32_t count) { return border.ties > before ? min(border.ties - before, count) : 0u; };
    const unsigned long long w = (tid < segments ? sh.sum[tid] : 0) + ties_kept(ties_before, n) * border_w;
    const unsigned long long through = block_prefix<unsigned long long>(w, sh.part_sum, lane, wave);
    if (tid == kThreads - 1) sh.before_sum = through;
    __syncthreads();
    const unsigned long long total = sh.before_sum;
    __syncthreads();
    // u outside [0, 1) draws the first or the last kept entry
    const double u = (double)a.uniform[rowi], goal = u * (double)total;
    const unsigned long long target = goal > 0.0 ? min((unsigned long long)fmin(goal, 9.2e18), total - 1) : 0;
    if (through > target && through - w <= target) {
        sh.found = tid;
        sh.before_sum = through - w;
        sh.before_count = ties_before;
    }
    __syncthreads();
    if (wave != 0) return;
    const int s = sh.found, i0 = 8 * (kWave * s + lane);
    float x[8];
    load8<TYPE>(r.at, i0, r.vocab, r.aligned, x);
    unsigned long long wj[8], mine = 0;
    uint32_t ties = 0;
    bool tie[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        weigh(x[j], wj[j], tie[j]);
        ties += tie[j];
    }
    uint32_t before = sh.before_count + wave_prefix<uint32_t>(ties, lane) - ties;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (tie[j]) wj[j] = before++ < border.ties ? border_w : 0;
        mine += wj[j];
    }
    unsigned long long cum = sh.before_sum + wave_prefix<unsigned long long>(mine, lane) - mine;
    int drawn = -1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        cum += wj[j];
        if (drawn < 0 && cum > target && cum - wj[j] <= target) drawn = i0 + j;
    }
    if (drawn >= 0) a.out[rowi] = drawn;  // one lane's
}

template <int TYPE>
void launch_sample(const SampleArgs& a, int rows, hipStream_t st) {
    hipLaunchKernelGGL(sample_rows_kernel<TYPE>, dim3((unsigned)rows), dim3(kThreads), 0, st, a);
}

}  // namespace
}  // namespace moss

using namespace moss;

MOSS_API int moss_sample_rows(const void* logits, int dtype, int rows, long long stride, int vocab, const void* uniform,
                              const void* temperature, float temperature_value, const void* top_k, int top_k_value,
                              const void* top_p, float top_p_value, const void* min_p, float min_p_value, void* out,
                              void* stream) {
    MOSS_CHECK_ARG(logits && uniform && out && rows > 0 && rows <= (1 << 21) && vocab > 0 && vocab <= (1 << 19) &&
                   stride >= vocab && dtype >= 0 && dtype <= 2);
    MOSS_CHECK_ARG(MOSS_ALIGNED(logits, dtype == 2 ? 4 : 2) && MOSS_ALIGNED(uniform, 4) && MOSS_ALIGNED(temperature, 4) &&
                   MOSS_ALIGNED(top_k, 4) && MOSS_ALIGNED(top_p, 4) && MOSS_ALIGNED(min_p, 4) && MOSS_ALIGNED(out, 8));
    const SampleArgs a{logits, stride, vocab, (const float*)uniform, (const float*)temperature, (const int*)top_k,
                       (const float*)top_p, (const float*)min_p, temperature_value, top_p_value, min_p_value, top_k_value,
                       (int64_t*)out};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0)
        launch_sample<0>(a, rows, st);
    else if (dtype == 1)
        launch_sample<1>(a, rows, st);
    else
        launch_sample<2>(a, rows, st);
    return moss_launch_status();
}
