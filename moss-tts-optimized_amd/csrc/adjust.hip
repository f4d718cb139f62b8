// Penalties for repeated tokens, biases and masks on rows of logits, before they are sampled.
//
// For entry v of a row with logit x, with the row's tokens so far h_0 .. h_{n-1}, of which the first `prompt` are the prompt:
//   said = v among h;  c = how often v is among h_prompt ..
//   said:   x <- x > 0 ? x / repetition : x repetition
//   c > 0:  x <- x - (c frequency + presence)
//   x <- x + bias, of the last of the row's (id, bias) pairs that names v
//   -inf where the row's mask has a 0 at bit v
// in fp32, rounded once to the logits' type.  Ids outside the row name nothing.
//
// What bounds it: the row's bytes in and out, and for few rows the chain launch, tokens, counts, logits.  128 rows of 151,936
// bf16 logits, in a graph over three inputs: a copy 14.0 us, with a mask 15.5, with up to 4096 tokens a row 21, all together 24
// (called one after another 23); 512 rows of 1024 with up to 400 tokens 4.8 (5.1).  Long rows are 1280 workgroups for 512 places, and
// the last chunk of each is a quarter full.  A workgroup takes a chunk of a row: it asks for the row's tokens and the chunk's logits and mask
// bits before it waits for any of them (34 -> 30 us), counts the tokens in its range in LDS, with integers (a count, a flag, the
// largest index of a pair), so that no order of the atomics shows, and then changes and writes its entries.  A row's
// tokens are read once for each of its chunks, from the cache: a chunk of 16384 entries with counts of 16 bits, two
// workgroups of 1024 threads a CU (30 -> 26 us against 8192 with counts of 32 and 512 threads, three a CU, where that only
// serves for 2^15 tokens and more, which 15 bits and a flag cannot count); a short row is one workgroup of 256 threads (6.1 ->
// 5.3 us for the 512).
#include "common.h"

namespace moss {
namespace {

constexpr int kAhead = 4;        // tokens of a thread on their way together
constexpr int kSmallRow = 2048;  // entries that one workgroup of 256 threads takes
constexpr int kNarrow = 1 << 15; // tokens that 15 bits count
typedef _Float16 f16_t;

struct AdjustArgs {
    const void* logits;
    void* out;
    long long stride, out_stride;
    int row0, rows, vocab, chunks;  // rows row0 .. row0 + rows - 1
    const void* tokens;
    long long token_row, token_step;  // elements
    int width;
    const int* lengths;
    const int* prompt;
    const float *repetition, *presence, *frequency;
    float repetition_v, presence_v, frequency_v;
    const int* bias_ids;
    const float* bias;
    long long bias_ids_stride, bias_stride;
    int biases;
    const uint32_t* mask;
    long long mask_stride;
};

template <int TYPE>
struct Logit;
template <>
struct Logit<0> {
    typedef uint16_t Bits;
    static __device__ __forceinline__ float value(Bits b) { return bf16_bits(b); }
    static __device__ __forceinline__ Bits bits(float x) { return f32_to_bf16(x); }
};
template <>
struct Logit<1> {
    typedef uint16_t Bits;
    static __device__ __forceinline__ float value(Bits b) { return (float)__builtin_bit_cast(f16_t, b); }
    static __device__ __forceinline__ Bits bits(float x) { return __builtin_bit_cast(Bits, (f16_t)x); }
};
template <>
struct Logit<2> {
    typedef uint32_t Bits;
    static __device__ __forceinline__ float value(Bits b) { return __uint_as_float(b); }
    static __device__ __forceinline__ Bits bits(float x) { return __float_as_uint(x); }
};

// Eight entries as they lie in memory.
template <int TYPE>
struct Group {
    u32x4_t w[TYPE == 2 ? 2 : 1];
    __device__ __forceinline__ typename Logit<TYPE>::Bits get(int i) const {
        if constexpr (TYPE == 2) return w[i / 4][i % 4];
        else return (uint16_t)(w[0][i / 2] >> (16 * (i & 1)));
    }
    __device__ __forceinline__ void set(int i, typename Logit<TYPE>::Bits b) {
        if constexpr (TYPE == 2) w[i / 4][i % 4] = b;
        else w[0][i / 2] = i & 1 ? (w[0][i / 2] & 0xffffu) | ((uint32_t)b << 16) : (w[0][i / 2] & 0xffff0000u) | b;
    }
};

// COUNT: bits of a count and its flag.
template <int TYPE, typename Token, int COUNT, int THREADS, int CHUNK>
__global__ __launch_bounds__(THREADS) void adjust_rows_kernel(AdjustArgs a) {
    typedef Logit<TYPE> L;
    typedef typename L::Bits Bits;
    constexpr int kThreads = THREADS, kChunk = CHUNK, kGroups = kChunk / 8 / kThreads;  // groups of 8 entries, a thread's
    constexpr int kCounts = kChunk * COUNT / 32, kPer = 32 / COUNT;                      // words of all counts, counts of a word
    constexpr uint32_t kPrompt = 1u << (COUNT - 1);  // said in the prompt; below it the count
    extern __shared__ uint32_t counts[];       // the tokens; then [kChunk] of 16 bits: the biases
    uint32_t* last = counts + (a.tokens ? kCounts : 0);  // two entries a word
    // Workgroups go round the XCDs one by one: of every eight rows each is given to one of them, so that its chunks find its
    // tokens in one cache.
    int row, chunk;
    const int tid = threadIdx.x, eight = blockIdx.x / (8 * a.chunks);
    if (8 * eight + 8 <= a.rows) {
        const int at = blockIdx.x - eight * 8 * a.chunks;
        row = 8 * eight + at % 8, chunk = at / 8;
    } else {
        row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    }
    row += a.row0;
    const Bits* src = reinterpret_cast<const Bits*>(a.logits) + (size_t)row * a.stride;
    Bits* dst = reinterpret_cast<Bits*>(a.out) + (size_t)row * a.out_stride;
    // Groups of eight entries that begin at 16 bytes (32 of fp32) in both rows, where both begin at the same place among
    // them; else one by one.  Entry 0 is entry `shift` of group 0.
    constexpr int kBytes = 8 * sizeof(Bits);
    const int shift = (int)((uintptr_t)src % kBytes / sizeof(Bits));
    const bool wide = (uintptr_t)src % kBytes == (uintptr_t)dst % kBytes;
    const int from = chunk * kChunk - shift;   // the chunk's first entry (below 0: none)
    const int e0 = max(from, 0), e1 = min(from + kChunk, a.vocab);
    Group<TYPE> x[kGroups];
    auto first_of = [&](int g) { return from + 8 * (g * kThreads + tid); };
    auto whole = [&](int e) { return wide && e >= 0 && e + 8 <= a.vocab; };
    // everything that memory has to be asked for, before anything is waited for, the tokens first: what is asked for later
    // comes later
    const Token* tokens = reinterpret_cast<const Token*>(a.tokens) + (long long)row * a.token_row;
    Token said[kAhead];
    int n = 0, prompt = 0;
    float rep = 1.f, pres = 0.f, freq = 0.f;
    if (a.tokens) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) said[j] = tokens[(long long)min(j * kThreads + tid, a.width - 1) * a.token_step];
        n = a.lengths ? min(max(a.lengths[row], 0), a.width) : a.width;
        prompt = a.prompt ? a.prompt[row] : 0;
        rep = a.repetition ? a.repetition[row] : a.repetition_v;
        pres = a.presence ? a.presence[row] : a.presence_v;
        freq = a.frequency ? a.frequency[row] : a.frequency_v;
    }
    const int* ids = a.bias_ids + (long long)row * a.bias_ids_stride;
    int named = a.bias ? ids[min(tid, a.biases - 1)] : -1;
    const uint32_t* mask = a.mask ? a.mask + (long long)row * a.mask_stride : nullptr;
    const int last_word = (a.vocab - 1) >> 5;
    uint32_t bits[kGroups][2];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int e = first_of(g);
        if (!whole(e)) continue;
#pragma unroll
        for (int i = 0; i < (TYPE == 2 ? 2 : 1); ++i) x[g].w[i] = reinterpret_cast<const u32x4_t*>(src + e)[i];
        if (mask) {
            bits[g][0] = mask[e >> 5];
            bits[g][1] = mask[min((e >> 5) + 1, last_word)];
        }
    }
    if (a.tokens || a.bias) {
        const int words = (a.tokens ? kCounts : 0) + (a.bias ? kChunk / 2 : 0);
        for (int i = 4 * tid; i < words; i += 4 * kThreads) *reinterpret_cast<u32x4_t*>(counts + i) = u32x4_t{0u, 0u, 0u, 0u};
        __syncthreads();
        if (a.tokens) {
            for (int i0 = 0; i0 < n; i0 += kAhead * kThreads) {
                if (i0)
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) said[j] = tokens[(long long)min(i0 + j * kThreads + tid, n - 1) * a.token_step];
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const int i = i0 + j * kThreads + tid;
                    if (i >= n || said[j] < e0 || said[j] >= e1) continue;
                    const int k = (int)said[j] - from, up = COUNT * (k % kPer);
                    if (i < prompt) atomicOr(counts + k / kPer, kPrompt << up);
                    else atomicAdd(counts + k / kPer, 1u << up);
                }
            }
        }
        // of two pairs that name one entry the later holds: the largest index + 1, in 16 bits, by compare and swap
        for (int i = tid; i < a.biases; i += kThreads) {
            if (i >= kThreads) named = ids[i];
            if (named < e0 || named >= e1) continue;
            uint32_t* at = last + (named - from) / 2;
            const int up = 16 * ((named - from) & 1);
            uint32_t old = *at;
            while (((old >> up) & 0xffffu) < (uint32_t)(i + 1)) {
                const uint32_t next = (old & ~(0xffffu << up)) | ((uint32_t)(i + 1) << up);
                const uint32_t seen = atomicCAS(at, old, next);
                if (seen == old) break;
                old = seen;
            }
        }
        __syncthreads();
    }
    const float* bias = a.bias + (long long)row * a.bias_stride;
    // entry e (from + k) with count word c and bias index b: changed, or as it was
    auto change = [&](Bits& v, uint32_t c, uint32_t b) {
        float y = L::value(v);
        if (c) y = y > 0.f ? y / rep : y * rep;
        if (c & ~kPrompt) y -= (float)(c & ~kPrompt) * freq + pres;
        if (b) y += bias[b - 1];
        v = L::bits(y);
    };
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int e = first_of(g), k = e - from;
        if (whole(e)) {
            if (a.tokens || a.bias) {
                u32x4_t c[COUNT / 16] = {}, b = {};
                uint32_t some = 0;
                if (a.tokens)
#pragma unroll
                    for (int i = 0; i < COUNT / 16; ++i) {
                        c[i] = *reinterpret_cast<const u32x4_t*>(counts + k / kPer + 4 * i);
                        some |= c[i][0] | c[i][1] | c[i][2] | c[i][3];
                    }
                if (a.bias) {
                    b = *reinterpret_cast<const u32x4_t*>(last + k / 2);
                    some |= b[0] | b[1] | b[2] | b[3];
                }
                if (some) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t ci = COUNT == 32 ? c[i / 4][i % 4] : (c[0][i / 2] >> (16 * (i & 1))) & 0xffffu;
                        const uint32_t bi = (b[i / 2] >> (16 * (i & 1))) & 0xffffu;
                        if (ci | bi) {
                            Bits v = x[g].get(i);
                            change(v, ci, bi);
                            x[g].set(i, v);
                        }
                    }
                }
            }
            if (mask) {
                const uint32_t kept = (uint32_t)((bits[g][0] | (uint64_t)bits[g][1] << 32) >> (e & 31));
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!(kept >> i & 1)) x[g].set(i, L::bits(-INFINITY));
            }
#pragma unroll
            for (int i = 0; i < (TYPE == 2 ? 2 : 1); ++i) reinterpret_cast<u32x4_t*>(dst + e)[i] = x[g].w[i];
        } else {
            // a row's ends, or all of a chunk whose rows begin at different places: one entry a lane
            for (int i = 0; i < 8; ++i) {
                const int at = wide ? e + i : from + g * 8 * kThreads + i * kThreads + tid;
                if (at < 0 || at >= a.vocab) continue;
                Bits v = src[at];
                const uint32_t ci = a.tokens ? counts[(at - from) / kPer] >> (COUNT * ((at - from) % kPer)) & (kPrompt | (kPrompt - 1)) : 0u;
                const uint32_t bi = a.bias ? (last[(at - from) / 2] >> (16 * ((at - from) & 1))) & 0xffffu : 0u;
                if (ci | bi) change(v, ci, bi);
                if (mask && !(mask[at >> 5] >> (at & 31) & 1)) v = L::bits(-INFINITY);
                dst[at] = v;
            }
        }
    }
}

template <int TYPE, typename Token, int COUNT, int THREADS, int CHUNK>
int launch_adjust(AdjustArgs a, hipStream_t st) {
    a.chunks = (a.vocab + 7 + CHUNK - 1) / CHUNK;  // a row that begins inside a group of eight has its last entries one further
    const size_t lds = (a.tokens ? COUNT / 8 * CHUNK : 0) + (a.bias ? 2 * CHUNK : 0);
    // a grid has fewer than 2^32 threads: whole eights of rows at a time, all of them but for 2^21 rows of two chunks and the like
    const int rows = a.rows, most = (int)(((1ll << 32) - 1) / THREADS / a.chunks) & ~7;
    for (a.row0 = 0; a.row0 < rows; a.row0 += a.rows) {
        a.rows = rows - a.row0 < most ? rows - a.row0 : most;
        hipLaunchKernelGGL((adjust_rows_kernel<TYPE, Token, COUNT, THREADS, CHUNK>), dim3((unsigned)a.rows * a.chunks), dim3(THREADS), lds,
                           st, a);
        if (const int status = moss_launch_status()) return status;
    }
    return 0;
}

template <int TYPE, typename Token>
int launch_adjust(const AdjustArgs& a, hipStream_t st) {
    if (a.vocab + 7 <= kSmallRow) return launch_adjust<TYPE, Token, 32, 256, kSmallRow>(a, st);
    return a.width < kNarrow ? launch_adjust<TYPE, Token, 16, 1024, 16384>(a, st) : launch_adjust<TYPE, Token, 32, 1024, 8192>(a, st);
}

template <int TYPE>
int launch_adjust(const AdjustArgs& a, int token_bytes, hipStream_t st) {
    return token_bytes == 8 ? launch_adjust<TYPE, int64_t>(a, st) : launch_adjust<TYPE, int32_t>(a, st);
}

}  // namespace
}  // namespace moss

using namespace moss;

MOSS_API int moss_adjust_rows(const void* logits, int dtype, int rows, long long stride, int vocab, const void* tokens,
                              int token_bytes, long long token_row_stride, long long token_stride, int width, const void* lengths,
                              const void* prompt, const void* repetition, float repetition_value, const void* presence,
                              float presence_value, const void* frequency, float frequency_value, const void* bias_ids,
                              long long bias_ids_stride, const void* bias, long long bias_stride, int biases, const void* mask,
                              long long mask_stride, void* out, long long out_stride, void* stream) {
    const int size = dtype == 2 ? 4 : 2;
    MOSS_CHECK_ARG(logits && out && dtype >= 0 && dtype <= 2 && rows > 0 && rows <= (1 << 21) && vocab > 0 && vocab <= (1 << 19) &&
                   (long long)rows * vocab <= (1ll << 38) && stride >= vocab && out_stride >= vocab && MOSS_ALIGNED(logits, size) && MOSS_ALIGNED(out, size));
    MOSS_CHECK_ARG(!tokens || ((token_bytes == 4 || token_bytes == 8) && MOSS_ALIGNED(tokens, token_bytes) && width > 0 && width <= (1 << 30) &&
                               token_row_stride >= 0 && token_stride >= 0));
    MOSS_CHECK_ARG(tokens || (!lengths && !prompt && !repetition && !presence && !frequency));
    MOSS_CHECK_ARG(MOSS_ALIGNED(lengths, 4) && MOSS_ALIGNED(prompt, 4) && MOSS_ALIGNED(repetition, 4) && MOSS_ALIGNED(presence, 4) &&
                   MOSS_ALIGNED(frequency, 4));
    const bool finite = repetition_value - repetition_value == 0.f && presence_value - presence_value == 0.f &&
                        frequency_value - frequency_value == 0.f;
    MOSS_CHECK_ARG(!tokens || (finite && (repetition || repetition_value > 0.f)));
    MOSS_CHECK_ARG((bias_ids == nullptr) == (bias == nullptr));
    MOSS_CHECK_ARG(!bias || (biases > 0 && biases < (1 << 16) && (bias_ids_stride == 0 || bias_ids_stride >= biases) &&
                             (bias_stride == 0 || bias_stride >= biases) && MOSS_ALIGNED(bias_ids, 4) && MOSS_ALIGNED(bias, 4)));
    MOSS_CHECK_ARG(!mask || ((mask_stride == 0 || mask_stride >= (vocab + 31) / 32) && MOSS_ALIGNED(mask, 4)));
    AdjustArgs a;
    a.logits = logits, a.out = out, a.stride = stride, a.out_stride = out_stride, a.row0 = 0, a.rows = rows, a.vocab = vocab;
    a.tokens = tokens, a.token_row = token_row_stride, a.token_step = token_stride, a.width = width;
    a.lengths = (const int*)lengths, a.prompt = (const int*)prompt;
    a.repetition = (const float*)repetition, a.presence = (const float*)presence, a.frequency = (const float*)frequency;
    a.repetition_v = repetition_value, a.presence_v = presence_value, a.frequency_v = frequency_value;
    a.bias_ids = (const int*)bias_ids, a.bias = (const float*)bias, a.bias_ids_stride = bias_ids_stride, a.bias_stride = bias_stride;
    a.biases = biases, a.mask = (const uint32_t*)mask, a.mask_stride = mask_stride;
    hipStream_t st = (hipStream_t)stream;
    return dtype == 0 ? launch_adjust<0>(a, token_bytes, st) : dtype == 1 ? launch_adjust<1>(a, token_bytes, st) : launch_adjust<2>(a, token_bytes, st);
}
