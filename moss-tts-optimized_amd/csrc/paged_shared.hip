// Attention of one new token per sequence over a paged cache, where sequences that stand next to each other in the batch share the
// first rows of their caches: those are read and multiplied once for all of them.
//
// o_h = sum_t softmax_t(scale q_h . k_t) v_t over the rows t < length, as paged_decode.hip has it.  A run is neighbouring
// sequences with the same group number (not below 0); runs end at every 64th sequence of the batch, so a wave sees
// whole ones.  With P the rows that a run's first sequence shares (at most its length, whole 16 rows), sequence b takes
// n_b = min(P, shared[b]), whole 16 rows, or all of its length if that is no more, from the pages of the first one, and the rest
// from its own.  A run of one shares nothing.
//
// The prefix: all of a run's query heads of a KV head are the rows of tiles, which go over the keys on the matrix cores
// (paged_prompt.h), row b up to key n_b; a tile's keys are cut into parts, so that few tiles fill the device.  The rest: paged_decode.h,
// from row n_b on.  Both leave (m, l, O), and a last launch joins a sequence's.  Who takes what is computed on the device by
// every wave from groups, shared and lengths, so that a captured graph follows them.
#include "paged_decode.h"
#include "paged_prompt.h"

namespace moss {
namespace {

constexpr int kPrefixTarget = 256;  // workgroups that the prefixes are shared out over

struct SharedArgs {
    DecodeArgs a;             // part and stat: of the sequences' own rows
    const int* groups;        // [B]
    const int* shared;        // [B]
    float* prefix_part;       // [KH, rows, D]
    float2* prefix_stat;      // [KH, rows]
    long long prefix_rows;
    int prefix_shares;
};

// Sequence b0 + lane of the batch: where its own rows begin, and its run.
struct Member {
    int length, from;  // its rows, of which the first `from` are the run's
    int first, size;   // the run's lanes
    int rows;          // P; 0 for a run of one
    __device__ __forceinline__ int own() const { return length - from; }
};

__device__ __forceinline__ Member member_of(const SharedArgs& s, const PagedBatch& bt, int shift, int b0, int lane) {
    const int b = b0 + lane;
    const bool in = b < bt.B;
    const int id = in ? s.groups[b] : -1, want = in ? max(s.shared[b], 0) : 0;
    Member m;
    m.length = in ? paged_length(bt, b, shift) : 0;
    const int before = __shfl_up(id, 1);
    const unsigned long long heads = __ballot(lane == 0 || id < 0 || id != before);
    const unsigned long long up_to = ~0ull >> (kWave - 1 - lane);
    m.first = kWave - 1 - __builtin_clzll(heads & up_to);
    const unsigned long long behind = heads & ~up_to;
    m.size = (behind ? __builtin_ctzll(behind) : kWave) - m.first;
    m.rows = m.size > 1 ? shared_rows(__shfl(want, m.first), __shfl(m.length, m.first)) : 0;
    m.from = shared_from(m.rows, want, m.length);
    return m;
}

// A run's tiles of `height` rows (of its first lane; 0 elsewhere), and their blocks of keys.
__device__ __forceinline__ int tiles_of(const Member& m, int group, int height, int lane) {
    return m.first == lane && m.rows > 0 ? (m.size * group + height - 1) / height : 0;
}
__device__ __forceinline__ int blocks_of(const Member& m) { return (m.rows + kPromptBlock - 1) / kPromptBlock; }

// What the batch's work is cut into: blocks of keys of a part of a prefix, units of a share of own rows, parts in all.  `at(b0)`
// gives the members from sequence b0 on.
struct Cuts {
    int share, units;
    long long items;
};
template <int HEIGHT, typename At>
__device__ __forceinline__ Cuts cuts_of(const SharedArgs& s, int B, int lane, At at) {
    long long blocks = 0, units = 0, items = 0;
    for (int b0 = 0; b0 < B; b0 += kWave) {
        const Member m = at(b0);
        blocks += (long long)tiles_of(m, s.a.group, HEIGHT, lane) * blocks_of(m);
        units += units_of(m.own());
    }
    Cuts c;
    c.share = prefix_share_of(wave_total(blocks), s.prefix_shares);
    c.units = share_of_units(wave_total(units), s.a.shares);
    for (int b0 = 0; b0 < B; b0 += kWave) {
        const Member m = at(b0);
        items += (long long)tiles_of(m, s.a.group, HEIGHT, lane) * shares_of(blocks_of(m), c.share);
    }
    c.items = wave_total(items);
    return c;
}

// One part of a run's prefix for a tile of its rows.
template <typename E, int D, int KS, typename S>
__device__ __forceinline__ void prefix_part(const SharedArgs& s, const typename S::Cache& c, const PagedBatch& bt, const Member& m, int b0,
                                            int l, int base, int index, int share, int kvh, Stage<D>& even, Stage<D>& odd) {
    constexpr int HEIGHT = 128 / KS, RW = 4 / KS, DT = D / 32, DK = D / 16;
    const DecodeArgs& a = s.a;
    const int lane = threadIdx.x & (kWave - 1), half = lane >> 5, rl = lane & 31, G = a.group;
    const int rw = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) % RW;
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int size = lane_value(m.size, l), P = lane_value(m.rows, l), blocks = (P + kPromptBlock - 1) / kPromptBlock;
    const int parts = shares_of(blocks, share), tile = uniform(index / parts), part = uniform(index % parts);
    const int nrows = size * G, row = min(tile * HEIGHT + 32 * rw + rl, nrows - 1);  // clamped: stores are guarded
    const int token = (int)((unsigned)row / (unsigned)G), head = kvh * G + row - token * G;
    TileRows rows;
    rows.qpos = __shfl(m.from, l + token) - 1;
    const int b = b0 + l;
    u32x4_t qf[DK];  // lane: row rl, dims 16 kk + 8 half .. + 7
    {
        const uint16_t* qr = a.q + (size_t)(b + token) * a.q_stride + (size_t)head * D + 8 * half;
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) qf[kk] = *reinterpret_cast<const u32x4_t*>(qr + 16 * kk) ^ a.flip;
    }
    int least = rows.qpos, most = rows.qpos;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        least = min(least, __shfl_xor(least, x));
        most = max(most, __shfl_xor(most, x));
    }
    rows.trow = bt.table + (size_t)b * bt.table_stride;
    rows.kvh = kvh, rows.b0 = part * share, rows.b1 = min(blocks, rows.b0 + share), rows.last = P - 1;
    rows.wave_first = uniform(least), rows.wave_last = uniform(most);
    rows.idle = tile * HEIGHT + 32 * rw >= nrows;
    f32x16_v o[DT];
    float mx, sum;
    if (!attend_rows<E, D, KS, S>(c, rows, bt.W, qf, a.scale, even, odd, o, mx, sum)) return;
    const int out = base + part * nrows + row;
    if (tile * HEIGHT + 32 * rw + rl >= nrows || !in_slots(out, 1, s.prefix_rows)) return;
    const size_t at = (size_t)kvh * s.prefix_rows + out;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<float4*>(s.prefix_part + at * D + 32 * dt + 8 * q4 + 4 * half) =
                make_float4(o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]);
    if (half == 0) s.prefix_stat[at] = make_float2(mx, sum);
}

// The parts of the prefixes (matrix cores) and the shares of the rest (memory) side by side in one launch, the parts first.
template <typename E, int D, int KS, typename S, typename T, bool NT>
__global__ __launch_bounds__(256, 2) void paged_shared_split(SharedArgs s, typename S::Cache c, PagedBatch bt) {
    constexpr int HEIGHT = 128 / KS;
    __shared__ __attribute__((aligned(1024))) Stage<D> even, odd;
    const DecodeArgs& a = s.a;
    const int lane = threadIdx.x & (kWave - 1), G = a.group;
    const Member m0 = member_of(s, bt, c.shift, 0, lane);
    auto at = [&](int b0) { return b0 == 0 ? m0 : member_of(s, bt, c.shift, b0, lane); };
    const Cuts cuts = cuts_of<HEIGHT>(s, bt.B, lane, at);
    const long long prefixes = cuts.items * c.kh;
    if (blockIdx.x < prefixes) {
        const int kvh = blockIdx.x % c.kh, item = blockIdx.x / c.kh;
        int before = 0, base = 0;
        for (int b0 = 0; b0 < bt.B; b0 += kWave) {
            const Member m = at(b0);
            const int tiles = tiles_of(m, G, HEIGHT, lane), parts = shares_of(blocks_of(m), cuts.share), n = tiles * parts;
            const int rows = tiles ? m.size * G * parts : 0;
            const int through = wave_prefix(n), rows_through = wave_prefix(rows);
            const unsigned long long past = __ballot(before + through > item);
            if (past) {
                const int l = __builtin_ctzll(past);
                prefix_part<E, D, KS, S>(s, c, bt, m, b0, l, base + lane_value(rows_through, l) - lane_value(rows, l),
                                         item - before - (lane_value(through, l) - lane_value(n, l)), cuts.share, kvh, even, odd);
                return;
            }
            before += lane_value(through, kWave - 1);
            base += lane_value(rows_through, kWave - 1);
        }
        return;
    }
    const int tiles = (G + 15) / 16, own = (int)(blockIdx.x - prefixes), slot = own / a.xdim, x = own % a.xdim;
    ShareOf sh;
    int before = 0;
    sh.b = -1;
    for (int b0 = 0; b0 < bt.B; b0 += kWave) {
        const Member m = at(b0);
        const int n = shares_of(units_of(m.own()), cuts.units), through = wave_prefix(n);
        const unsigned long long past = __ballot(before + through > slot);
        if (past) {
            const int l = __builtin_ctzll(past), count = lane_value(n, l), from = lane_value(m.from, l);
            sh.b = b0 + l;
            share_rows(lane_value(m.length, l) - from, count, slot - before - (lane_value(through, l) - count), sh.r0, sh.r1);
            sh.r0 += from, sh.r1 += from;
            sh.alone = count == 1 && from == 0;
            break;
        }
        before += lane_value(through, kWave - 1);
    }
    if (sh.b < 0 || slot >= a.slots) return;
    sh.kvh = x / tiles, sh.h0 = 16 * (x % tiles), sh.heads = min(16, G - sh.h0), sh.slot = slot;
    static_assert(sizeof(float[4][16][D]) <= sizeof(Stage<D>) && 2 * sizeof(float[4][16]) <= sizeof(Stage<D>), "");
    float(&ml)[2][4][16] = *reinterpret_cast<float(*)[2][4][16]>(odd);
    decode_share<E, D, T, NT>(a, c, bt, sh, *reinterpret_cast<float(*)[4][16][D]>(even), ml[0], ml[1]);
}

// grid (QH, B), 256 threads: the parts of the prefix and the shares of the rest of one head of a sequence, wave w taking w, w + 4,
// ..; the four waves' sums meet in LDS.
template <typename E, int D, int HEIGHT>
__global__ __launch_bounds__(256) void paged_shared_join(SharedArgs s, int shift, PagedBatch bt) {
    constexpr int VPL = D / kWave;
    __shared__ float acc_s[4][D];
    const DecodeArgs& a = s.a;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & (kWave - 1), w = tid / kWave, G = a.group;
    const int mine = b % kWave;
    const Member m0 = member_of(s, bt, shift, 0, lane);
    auto at = [&](int b0) { return b0 == 0 ? m0 : member_of(s, bt, shift, b0, lane); };
    const Cuts cuts = cuts_of<HEIGHT>(s, bt.B, lane, at);
    const int share = cuts.share, su = cuts.units;
    // partial results before this sequence's, and its run
    Member m;
    int slots = 0, rows = 0;
    for (int b0 = 0;; b0 += kWave) {
        m = at(b0);
        const int n = shares_of(units_of(m.own()), su);
        const int r = tiles_of(m, G, HEIGHT, lane) ? m.size * G * shares_of(blocks_of(m), share) : 0;
        if (b0 + kWave > b) {
            const int l = lane_value(m.first, mine);
            slots += wave_total(lane < mine ? n : 0);
            rows += wave_total(lane < l ? r : 0);
            break;
        }
        slots += wave_total(n);
        rows += wave_total(r);
    }
    const int own = shares_of(units_of(lane_value(m.own(), mine)), su), from = lane_value(m.from, mine);
    const int parts = from > 0 ? shares_of((lane_value(m.rows, mine) + kPromptBlock - 1) / kPromptBlock, share) : 0;
    if (parts == 0 && own == 1) return;  // written by its workgroup
    uint16_t* dst = a.out + ((size_t)b * a.qh + h) * D;
    const int count = parts + own;
    if (count == 0) {
        for (int d = tid; d < D; d += 256) dst[d] = 0;
        return;
    }
    const int first = lane_value(m.first, mine), nrows = lane_value(m.size, mine) * G;
    const int row = rows + (mine - first) * G + h % G;
    // only when what says where rows are changes between the launches
    if (!in_slots(slots, own, a.slots) || (parts && !in_slots(row, (parts - 1) * nrows + 1, s.prefix_rows))) return;
    // part i's place among the statistics and results: the prefix's, then the sequence's own
    const size_t step = nrows;
    const float2* stat0 = s.prefix_stat + (size_t)(h / G) * s.prefix_rows + row;
    const float2* stat1 = a.stat + (size_t)slots * a.qh + h;
    const float* part0 = s.prefix_part + ((size_t)(h / G) * s.prefix_rows + row) * D;
    const float* part1 = a.part + ((size_t)slots * a.qh + h) * D;
    auto stat = [&](int i) { return i < parts ? stat0[i * step] : stat1[(size_t)(i - parts) * a.qh]; };
    auto part = [&](int i) { return i < parts ? part0 + i * step * D : part1 + (size_t)(i - parts) * a.qh * D; };
    const float2 mls = lane < count ? stat(lane) : make_float2(-INFINITY, 0.f);
    float mx = mls.x;
    for (int i = kWave + lane; i < count; i += kWave) mx = fmaxf(mx, stat(i).x);
    mx = wave_max(mx);
    auto weight = [&](float v) { return v == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v - mx); };
    const float f0 = weight(mls.x);
    float den = f0 * mls.y;
    for (int i = kWave + lane; i < count; i += kWave) {
        const float2 v = stat(i);
        den += weight(v.x) * v.y;
    }
    den = wave_sum(den);
    float acc[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] = 0.f;
    constexpr int N = 8;  // parts on their way together: w, w + 4, ..
    for (int s0 = w; s0 < count; s0 += 4 * N) {
        float x[N][VPL], f[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float* p = part(min(s0 + 4 * n, count - 1)) + VPL * lane;
#pragma unroll
            for (int i = 0; i < VPL; ++i) x[n][i] = p[i];
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = min(s0 + 4 * n, count - 1);
            f[n] = i < kWave ? __uint_as_float(lane_value(__float_as_uint(f0), i)) : weight(stat(i).x);
            if (s0 + 4 * n >= count) f[n] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < VPL; ++i) acc[i] = f[n] == 0.f ? acc[i] : fmaf(f[n], x[n][i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc_s[w][VPL * lane + i] = acc[i];
    __syncthreads();
    if (tid < D / 2) {
        const float inv = den == 0.f ? 0.f : 1.0f / den;
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            x += acc_s[v][2 * tid];
            y += acc_s[v][2 * tid + 1];
        }
        reinterpret_cast<uint32_t*>(dst)[tid] = E::pack(x * inv, y * inv);
    }
}

struct SharedPlan {
    int xdim, shares, prefix_shares;
    long long slots, rows, items;  // of the prefixes: rows of partial results, workgroups a KV head at most
    int height;
};

SharedPlan shared_plan(int B, int W, int shift, int qh, int kh) {
    SharedPlan p;
    const long long G = qh / kh;
    p.xdim = kh * (int)((G + 15) / 16);
    p.shares = kTarget / p.xdim > 1 ? kTarget / p.xdim : 1;
    p.slots = decode_slots(B, W, shift, p.shares);
    p.prefix_shares = kPrefixTarget / kh > 1 ? kPrefixTarget / kh : 1;
    p.height = B * G * kh <= 1024 ? 64 : 128;
    prefix_bounds(B, (int)G, p.height, p.prefix_shares, p.items, p.rows);
    return p;
}

template <typename E, int D, int KS, typename T, typename S>
int launch_shared(const SharedArgs& s, const typename S::Cache& c, const PagedBatch& bt, const SharedPlan& p, hipStream_t st) {
    const long long blocks = p.items * c.kh + p.slots * p.xdim;
    MOSS_CHECK_ARG(blocks * 256 < (1ll << 32));
    const long long page = ((long long)c.kh << c.shift) * D * (std::is_same<typename S::Cache, PagedCache>::value ? 2 : 1);
    const long long named = (long long)bt.B * bt.W;
    if ((named < c.pages ? named : c.pages) * page * 2 > kCached)
        hipLaunchKernelGGL((paged_shared_split<E, D, KS, S, T, true>), dim3((unsigned)blocks), dim3(256), 0, st, s, c, bt);
    else
        hipLaunchKernelGGL((paged_shared_split<E, D, KS, S, T, false>), dim3((unsigned)blocks), dim3(256), 0, st, s, c, bt);
    hipLaunchKernelGGL((paged_shared_join<E, D, 128 / KS>), dim3((unsigned)s.a.qh, (unsigned)bt.B), dim3(256), 0, st, s, c.shift, bt);
    return moss_launch_status();
}

template <typename E, int D, template <typename, int> class T, template <typename, int> class S, typename Cache>
int launch_shared(const SharedArgs& s, const Cache& c, const PagedBatch& bt, const SharedPlan& p, hipStream_t st) {
    return p.height == 64 ? launch_shared<E, D, 2, T<E, D>, S<E, D>>(s, c, bt, p, st) : launch_shared<E, D, 1, T<E, D>, S<E, D>>(s, c, bt, p, st);
}

long long workspace_bytes_of(const SharedPlan& p, int qh, int kh, int d) { return (p.slots * qh + p.rows * kh) * (d + 2) * 4; }

template <template <typename, int> class T, template <typename, int> class S, typename Cache>
int shared_decode(const void* q, long long q_stride, const Cache& c, const PagedBatch& bt, const void* groups, const void* shared,
                  int qh, int d, float scale, void* out, void* workspace, long long workspace_bytes, int dtype, void* stream) {
    MOSS_CHECK_ARG(q && out && workspace && groups && shared && paged_pointers_ok(c, bt) && paged_shape_ok(c, bt, qh, d));
    MOSS_CHECK_ARG((dtype == 0 || dtype == 1) && q_stride % 8 == 0 && q_stride >= (long long)qh * d && scale == scale);
    MOSS_CHECK_ARG(MOSS_ALIGNED(q, 16) && MOSS_ALIGNED(out, 16) && MOSS_ALIGNED(workspace, 16) && MOSS_ALIGNED(groups, 4) &&
                   MOSS_ALIGNED(shared, 4));
    const SharedPlan p = shared_plan(bt.B, bt.W, c.shift, qh, c.kh);
    MOSS_CHECK_ARG(workspace_bytes >= workspace_bytes_of(p, qh, c.kh, d));
    const long long own = p.slots * qh, rows = p.rows * c.kh;
    float* part = (float*)workspace;
    float* prefix_part = part + own * d;
    float2* stat = reinterpret_cast<float2*>(prefix_part + rows * d);
    // the scale is positive in either half, its sign goes to q; never 0, so a masked score stays -inf
    const DecodeArgs a{(const uint16_t*)q, q_stride, (uint16_t*)out, part, stat, qh, qh / c.kh, p.xdim, p.shares, p.slots,
                       fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f), scale < 0.f ? 0x80008000u : 0u};
    const SharedArgs s{a, (const int*)groups, (const int*)shared, prefix_part, stat + own, p.rows, p.prefix_shares};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0)
        return d == 128 ? launch_shared<Bf16, 128, T, S>(s, c, bt, p, st) : launch_shared<Bf16, 64, T, S>(s, c, bt, p, st);
    return d == 128 ? launch_shared<F16, 128, T, S>(s, c, bt, p, st) : launch_shared<F16, 64, T, S>(s, c, bt, p, st);
}

}  // namespace
}  // namespace moss

using namespace moss;

MOSS_API long long moss_paged_shared_workspace_bytes(int B, int W, int page_rows, int qh, int kh, int d) {
    const int shift = page_shift(page_rows);
    if (B <= 0 || B > 65535 || W <= 0 || shift < 0 || ((long long)W << shift) > (1ll << 30) || kh <= 0 || qh <= 0 || qh % kh ||
        qh > 1024 || (d != 64 && d != 128))
        return 0;
    return workspace_bytes_of(shared_plan(B, W, shift, qh, kh), qh, kh, d);
}

MOSS_API int moss_paged_shared_decode_attention(const void* q, long long q_stride, const void* k, const void* v, long long k_stride,
                                                long long v_stride, int pages, int page_rows, const void* table,
                                                long long table_stride, const void* lengths, const void* groups,
                                                const void* shared, int B, int W, int qh, int kh, int d, float scale, void* out,
                                                void* workspace, long long workspace_bytes, int dtype, void* stream) {
    const PagedCache c = paged_cache(k, v, k_stride, v_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, nullptr, B, W, table_stride};
    return shared_decode<Tile16, Stage16>(q, q_stride, c, bt, groups, shared, qh, d, scale, out, workspace, workspace_bytes, dtype, stream);
}

MOSS_API int moss_paged_shared_decode_attention_fp8(const void* q, long long q_stride, const void* k, const void* v,
                                                    const void* k_scales, const void* v_scales, long long k_stride,
                                                    long long v_stride, long long k_scale_stride, long long v_scale_stride,
                                                    int pages, int page_rows, const void* table, long long table_stride,
                                                    const void* lengths, const void* groups, const void* shared, int B, int W,
                                                    int qh, int kh, int d, float scale, void* out, void* workspace,
                                                    long long workspace_bytes, int dtype, void* stream) {
    const PagedCache8 c = paged_cache8(k, v, k_scales, v_scales, k_stride, v_stride, k_scale_stride, v_scale_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, nullptr, B, W, table_stride};
    MOSS_CHECK_ARG(paged8_ok(c));
    return shared_decode<Tile8, Stage8>(q, q_stride, c, bt, groups, shared, qh, d, scale, out, workspace, workspace_bytes, dtype, stream);
}
