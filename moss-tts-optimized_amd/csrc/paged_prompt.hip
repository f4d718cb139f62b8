// Causal attention of packed prompts over a paged cache, on the matrix cores.
//
// The T packed tokens belong to B sequences (starts[b] .. starts[b + 1] - 1); token i of a sequence's n stands at
// position length - n + i and attends the rows 0 .. position of its sequence's pages, the cached ones before it and
// the new ones up to itself (all written).  o_h = sum_t softmax_t(scale q_h . k_t) v_t with query head h reading KV head
// h / (QH / KH); a token without a visible row gives zeros; tokens behind the last sequence are left alone.
//
// Work: the rows of a tile are (token, query head of the KV head's group) pairs, token first, so any group size fills
// them.  A workgroup takes 128 rows of one sequence and KV head, a wave 32 of them, over all keys or, where a tile sees
// many more than a workgroup's fair share of the whole call (a few new tokens behind a long prefix), over a part of them:
// such parts leave (m, l, O) in a workspace, and a second launch joins them.  Who takes what follows from starts and lengths
// on the device (paged_index.h).
// A wave's part of it is in paged_prompt.h.
// What bounds it: the matrix and vector pipes in turn at the clock that power holds (8000 tokens of 32 / 8 heads of 128:
// 520 to 550 us, 950 to 1010 TFLOP/s, where a large product of bf16 matrices reaches 1640); with K and V through registers, V
// transposed on the way, 667 us.  From 8 bits 572 us beside 539: the conversion of a block, once a workgroup, is 19 of 137 million
// vector instructions (118 from 16 bits), and the matrix pipes are as busy; six registers of the whole tiles' kernel for heads of
// 128 are spilled.  Heads of 64, whole tiles, have two waves a SIMD from 8 bits (174 to 187 registers) and three from 16: 8000 tokens
// of 12 / 12 heads 149 us from 8 bits and 162 from 16, of 16 / 2 heads 197 and 192; 2500 tokens 38 and 33.
#include "paged_prompt.h"

namespace moss {
namespace {

struct PromptArgs {
    const uint16_t* q;
    long long q_stride;
    uint16_t* out;
    float* part;   // [slots, KH, D / 4, 128 rows] of 4: O of each part
    float2* stat;  // [slots, KH, 128]: its m and l
    int T, qh, group, shares;
    long long slots;
    float scale;    // |scale| log2(e), not 0: a masked score stays -inf
    uint32_t flip;  // its sign, for the two values of a word of q
};

// A workgroup's sequence and its item's number, of what count(tiles, share) counts; `first`: partial results of the
// sequences taken before it.  A batch of up to 64 is one read of lengths and starts, and taken in the order of its lengths.
struct Found {
    PromptTiles tiles;
    int b, tok0, index, share, first;  // b -1: none
};
template <int HEIGHT, typename Count>
__device__ __forceinline__ Found find_tile(const PromptArgs& a, int shift, const PagedBatch& bt, int item, int lane,
                                           Count count) {
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };  // it is; this puts it into a scalar
    auto of = [&](int b, int& tok0) {
        const int2 t = paged_tokens(bt, b, a.T);
        tok0 = t.x;
        return PromptTiles{t.y, a.group, paged_length(bt, b, shift) - t.y, HEIGHT};
    };
    auto parts = [&](const PromptTiles& t, int share) { return t.tiles_over(share) ? t.parts(share) : 0; };
    Found f;
    int tok0 = 0;
    if (bt.B <= kWave) {
        PromptTiles t{0, a.group, 0, HEIGHT};
        int b = lane;
        if (lane < bt.B) t = of(lane, tok0);
        if (bt.B > 1) {
            // longest first: its tiles see the most keys, and what is taken last ends last.  (Nine prompts that come shortest
            // first 64 -> 48 us.)
            const int key = lane < bt.B ? (t.pos0 + t.tokens) / kPromptBlock * kWave + kWave - 1 - lane : -1;
            int place = 0;
            for (int j0 = 0; j0 < bt.B; j0 += 8)
#pragma unroll
                for (int j = 0; j < 8; ++j) place += __builtin_amdgcn_readlane(key, j0 + j) > key;
            if (lane >= bt.B) place = lane;
            auto move = [&](int v) { return __builtin_amdgcn_ds_permute(4 * place, v); };
            b = move(b);
            tok0 = move(tok0);
            t = PromptTiles{move(t.tokens), a.group, move(t.pos0), HEIGHT};
        }
        f.share = uniform(prompt_share(wave_total(t.blocks_bound()), a.shares));
        const int n = count(t, f.share), through = wave_prefix(n);
        const unsigned long long past = __ballot(through > item);
        f.b = -1;
        if (!past) return f;
        const int l = __builtin_ctzll(past);
        f.b = lane_value(b, l);
        f.tiles = PromptTiles{lane_value(t.tokens, l), a.group, lane_value(t.pos0, l), HEIGHT};
        f.tok0 = lane_value(tok0, l);
        f.index = item - (lane_value(through, l) - lane_value(n, l));
        f.first = wave_total(lane < l ? parts(t, f.share) : 0);
        return f;
    }
    long long blocks = 0;
    for (int b = lane; b < bt.B; b += kWave) blocks += of(b, tok0).blocks_bound();
    f.share = uniform(prompt_share(wave_total(blocks), a.shares));
    const Place pl = find_item(bt.B, item, lane, [&](int b) { return count(of(b, tok0), f.share); });
    f.b = uniform(pl.b);
    if (f.b < 0) return f;
    const PromptTiles t = of(f.b, tok0);
    f.tiles = PromptTiles{uniform(t.tokens), a.group, uniform(t.pos0), HEIGHT};
    f.tok0 = uniform(tok0);
    f.index = uniform(pl.index);
    int before = 0;
    for (int s = lane; s < f.b; s += kWave) before += parts(of(s, tok0), f.share);
    f.first = wave_total(before);
    return f;
}

template <typename E, int D, int KS, typename S>
__global__ __launch_bounds__(256, 2) void paged_prompt_kernel(PromptArgs a, typename S::Cache c, PagedBatch bt) {
    constexpr int RW = 4 / KS, HEIGHT = 32 * RW, DT = D / 32, DK = D / 16;  // row waves
    __shared__ __attribute__((aligned(1024))) Stage<D> even, odd;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, rl = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rw = wave % RW;
    const int kvh = blockIdx.x % c.kh, G = a.group;  // neighbours in the grid, which lie on different XCDs, differ in it
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const Found f = find_tile<HEIGHT>(a, c.shift, bt, (int)(blockIdx.x / c.kh), lane,
                                      [](const PromptTiles& t, int s) { return t.items(s); });
    if (f.b < 0) return;
    const PromptTiles& tiles = f.tiles;
    const int share = f.share, tok0 = f.tok0, pos0 = tiles.pos0;
    const PromptItem found = prompt_item(tiles, share, f.index);
    const PromptItem item{uniform(found.tile), uniform(found.part), uniform(found.slot)};
    if (!is_item(tiles, share, item)) return;  // only when starts or lengths change under the kernel
    const int row0 = item.tile * HEIGHT, nrows = tiles.rows();
    const int row = min(row0 + 32 * rw + rl, nrows - 1);  // this lane's row (clamped: stores are guarded)
    const int token = tiles.token_of(row), head = kvh * G + row - token * G;
    const int qpos = pos0 + token;  // sees keys 0 .. qpos
    const int last = uniform(tiles.last_key(item.tile)), blocks = uniform(tiles.blocks(item.tile));  // the workgroup's last key
    const bool cut = blocks > share, idle = row0 + 32 * rw >= nrows;             // idle: no row of this wave's exists
    const int wave_last = uniform(pos0 + tiles.token_of(min(row0 + 32 * rw + 31, nrows - 1)));
    const int wave_first = uniform(pos0 + tiles.token_of(min(row0 + 32 * rw, nrows - 1)));  // keys up to it are seen by all its rows
    const int b0 = uniform(item.part * share), b1 = uniform(min(blocks, b0 + share));

    u32x4_t qf[DK];  // lane: row rl, dims 16 kk + 8 half .. + 7
    {
        const uint16_t* qr = a.q + (size_t)(tok0 + token) * a.q_stride + (size_t)head * D + 8 * half;
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) qf[kk] = *reinterpret_cast<const u32x4_t*>(qr + 16 * kk) ^ a.flip;
    }
    f32x16_v o[DT];
    float m, l;
    const TileRows rows{bt.table + (size_t)f.b * bt.table_stride, kvh, b0, b1, last, qpos, wave_first, wave_last, idle};
    if (!attend_rows<E, D, KS, false, S>(c, rows, bt.W, qf, a.scale, tid, even, odd, o, m, l)) return;
    // O^T element e of d tile dt: d = 32 dt + 8 (e / 4) + 4 half + e % 4
    if (cut) {
        // (starts that do not rise can name more parts than there are tokens for: they have no slot)
        if (row0 + 32 * rw + rl >= nrows || !in_slots(f.first + item.slot, 1, a.slots)) return;
        const size_t at = (size_t)(f.first + item.slot) * c.kh + kvh;
        float4* part = reinterpret_cast<float4*>(a.part) + at * (D / 4) * HEIGHT + 32 * rw + rl;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                part[(8 * dt + 2 * q4 + half) * HEIGHT] =
                    make_float4(o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]);
        if (half == 0) a.stat[at * HEIGHT + 32 * rw + rl] = make_float2(m, l);
        return;
    }
    if (row0 + 32 * rw + rl >= nrows) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    uint16_t* dst = a.out + ((size_t)(tok0 + token) * a.qh + head) * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<uint2*>(dst + 32 * dt + 8 * q4 + 4 * half) =
                make_uint2(E::pack(o[dt][4 * q4] * inv, o[dt][4 * q4 + 1] * inv),
                           E::pack(o[dt][4 * q4 + 2] * inv, o[dt][4 * q4 + 3] * inv));
}

// The parts of one cut tile and KV head, two threads a row: thread (row, h) takes its 4-dim pieces h, h + 2, ..
template <typename E, int D, int HEIGHT>
__global__ __launch_bounds__(2 * HEIGHT) void paged_prompt_join(PromptArgs a, int kh, int shift, PagedBatch bt) {
    const int lane = threadIdx.x & 63, r = threadIdx.x % HEIGHT, h = threadIdx.x / HEIGHT, kvh = blockIdx.x % kh, G = a.group;
    const Found f = find_tile<HEIGHT>(a, shift, bt, (int)(blockIdx.x / kh), lane,
                                      [](const PromptTiles& t, int s) { return t.tiles_over(s); });
    if (f.b < 0) return;
    const int tile = f.tiles.tiles() - 1 - f.index, row = tile * HEIGHT + r;
    const int count = (f.tiles.blocks(tile) + f.share - 1) / f.share;
    if (tile < 0 || row >= f.tiles.rows()) return;  // (tile: as for an item)
    // part k's slot: the cut tiles' parts 0 come first, then those of the tiles of more than 1, 2, .. shares
    float m = -INFINITY, den = 0.f;
    float4 acc[D / 8];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    int slot = f.first + f.index;
    for (int k = 0; k < count && in_slots(slot, 1, a.slots); ++k) {
        const size_t at = ((size_t)slot * kh + kvh) * HEIGHT + r;
        slot += f.tiles.tiles_over(k ? k * f.share : f.share);
        const float2 st = a.stat[at];
        const float4* part = reinterpret_cast<const float4*>(a.part) + (at - r) * (D / 4) + r;
        float4 v[D / 8];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) v[i] = part[(2 * i + h) * HEIGHT];
        const float mn = fmaxf(m, st.x);
        const float f0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        const float f1 = st.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.x - mn);
        m = mn;
        den = den * f0 + st.y * f1;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            acc[i].x = acc[i].x * f0 + v[i].x * f1;
            acc[i].y = acc[i].y * f0 + v[i].y * f1;
            acc[i].z = acc[i].z * f0 + v[i].z * f1;
            acc[i].w = acc[i].w * f0 + v[i].w * f1;
        }
    }
    const float inv = den == 0.f ? 0.f : 1.0f / den;
    const int token = f.tiles.token_of(row);
    uint16_t* dst = a.out + ((size_t)(f.tok0 + token) * a.qh + kvh * G + row - token * G) * D;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<uint2*>(dst + 4 * (2 * i + h)) =
            make_uint2(E::pack(acc[i].x * inv, acc[i].y * inv), E::pack(acc[i].z * inv, acc[i].w * inv));
}

// Rows of a tile, tiles at most, shares of a KV head, partial results at most (0: no tile can see more than a share's
// least blocks).
struct PromptPlan {
    int height;
    long long tiles, slots;
    int shares;
};
// Tiles of 128 rows are halved, and the waves of a row share its keys, while there are few.  0 / 1024: 18.7 / 15.0 us for 512
// tokens of 32 / 8 heads, 7.7 / 6.9 for 45, 49.4 / 46.0 for nine prompts of 2800; 56.8 / 58.1 for 2048 tokens, 528 / 641
// (if it did) for 8000.
constexpr int kSmallTiles = 1024;
// From a cache in 8 bits, where halved tiles convert every block of keys twice as often, up to 512.  Halved / not: 9.6 / 10.7 us for
// 45 tokens, 20.2 / 24.9 for 512, 34.0 / 37.6 for 1024 (256 tiles), 73.0 / 71.6 for 2048 (512), 104 / 89 for 2500, 216 / 174 for
// 4096 (1024), 59.2 / 59.1 for the nine prompts (700), 40.9 / 34.4 for twelve of 260 (780).
constexpr int kSmallTiles8 = 512;
// Parts of the whole call's work, over all KV heads, that a tile is not cut below.  128 / 256 / 512: 29 / 22 / 23 us for 150
// tokens after 1900, 61 / 46 / 47 for 32 single tokens after 50 to 4000, 46 / 46 / 49 for the nine prompts.  (All from 16 bits, in
// halved tiles.  Whole ones of the nine prompts from 8 bits are 95 parts a KV head of up to 25 blocks, where 10.5 are even.)
constexpr int kShares = 256;

PromptPlan prompt_plan(int B, int W, int shift, int T, int qh, int kh, int small_tiles) {
    PromptPlan p;
    const long long rows = (long long)T * (qh / kh);
    p.height = (rows + 127) / 128 * kh <= small_tiles ? 64 : 128;
    p.tiles = (rows + p.height - 1) / p.height + (B < T ? B : T);
    p.shares = kShares / kh > 1 ? kShares / kh : 1;
    const long long parts = (((long long)W << shift) + kPromptShare * kPromptBlock - 1) / (kPromptShare * kPromptBlock);
    p.slots = parts <= 1 ? 0 : p.tiles * parts < 2 * p.shares ? p.tiles * parts : 2 * p.shares;
    return p;
}

long long workspace_bytes_of(const PromptPlan& p, int kh, int d) { return p.slots * kh * p.height * (d + 2) * 4; }

long long workspace_bytes_for(int B, int W, int page_rows, int T, int qh, int kh, int d, int small_tiles) {
    const int shift = page_shift(page_rows);
    if (B <= 0 || W <= 0 || shift < 0 || ((long long)W << shift) > (1ll << 30) || T <= 0 || kh <= 0 || qh <= 0 || qh % kh ||
        (d != 64 && d != 128))
        return 0;
    return workspace_bytes_of(prompt_plan(B, W, shift, T, qh, kh, small_tiles), kh, d);
}

template <typename E, int D, int KS, typename S>
int launch_prompt(const PromptArgs& a, const typename S::Cache& c, const PagedBatch& bt, const PromptPlan& p, hipStream_t st) {
    constexpr int HEIGHT = 128 / KS;
    const long long groups = (p.tiles + (p.slots ? p.shares : 0)) * c.kh;
    MOSS_CHECK_ARG(groups * 256 < (1ll << 32));
    hipLaunchKernelGGL((paged_prompt_kernel<E, D, KS, S>), dim3((unsigned)groups), dim3(256), 0, st, a, c, bt);
    if (p.slots) {
        const long long cut = (p.tiles < p.shares ? p.tiles : p.shares) * c.kh;
        hipLaunchKernelGGL((paged_prompt_join<E, D, HEIGHT>), dim3((unsigned)cut), dim3(2 * HEIGHT), 0, st, a, c.kh, c.shift, bt);
    }
    return moss_launch_status();
}

template <typename E, int D, typename S>
int launch_prompt(const PromptArgs& a, const typename S::Cache& c, const PagedBatch& bt, const PromptPlan& p, hipStream_t st) {
    return p.height == 64 ? launch_prompt<E, D, 2, S>(a, c, bt, p, st) : launch_prompt<E, D, 1, S>(a, c, bt, p, st);
}

template <template <typename, int> class S, typename Cache>
int prompt(const void* q, long long q_stride, const Cache& c, const PagedBatch& bt, int T, int qh, int d, float scale, void* out,
           void* workspace, long long workspace_bytes, int dtype, void* stream) {
    MOSS_CHECK_ARG(q && out && bt.starts && paged_pointers_ok(c, bt) && paged_shape_ok(c, bt, qh, d));
    MOSS_CHECK_ARG((dtype == 0 || dtype == 1) && T > 0 && T <= (1 << 20) && q_stride % 8 == 0 &&
                   q_stride >= (long long)qh * d && paged_scale_ok(scale));
    MOSS_CHECK_ARG(MOSS_ALIGNED(q, 16) && MOSS_ALIGNED(out, 16) && MOSS_ALIGNED(workspace, 16));
    PromptPlan p = prompt_plan(bt.B, bt.W, c.shift, T, qh, c.kh, std::is_same<Cache, PagedCache8>::value ? kSmallTiles8 : kSmallTiles);
    // whole tiles' parts need up to twice the halved ones': a workspace of the 16-bit form's size serves with those
    if (workspace && workspace_bytes < workspace_bytes_of(p, c.kh, d)) p = prompt_plan(bt.B, bt.W, c.shift, T, qh, c.kh, kSmallTiles);
    MOSS_CHECK_ARG(p.slots == 0 || (workspace && workspace_bytes >= workspace_bytes_of(p, c.kh, d)));
    const long long values = p.slots * c.kh * p.height;
    const PromptArgs a{(const uint16_t*)q, q_stride, (uint16_t*)out, (float*)workspace,
                       reinterpret_cast<float2*>((float*)workspace + values * d), T, qh, qh / c.kh, p.shares,
                       p.slots, fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f), scale < 0.f ? 0x80008000u : 0u};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0)
        return d == 128 ? launch_prompt<Bf16, 128, S<Bf16, 128>>(a, c, bt, p, st) : launch_prompt<Bf16, 64, S<Bf16, 64>>(a, c, bt, p, st);
    return d == 128 ? launch_prompt<F16, 128, S<F16, 128>>(a, c, bt, p, st) : launch_prompt<F16, 64, S<F16, 64>>(a, c, bt, p, st);
}

}  // namespace
}  // namespace moss

using namespace moss;

MOSS_API long long moss_paged_prompt_workspace_bytes(int B, int W, int page_rows, int T, int qh, int kh, int d) {
    return workspace_bytes_for(B, W, page_rows, T, qh, kh, d, kSmallTiles);
}

MOSS_API long long moss_paged_prompt_workspace_bytes_fp8(int B, int W, int page_rows, int T, int qh, int kh, int d) {
    return workspace_bytes_for(B, W, page_rows, T, qh, kh, d, kSmallTiles8);
}

MOSS_API int moss_paged_prompt_attention(const void* q, long long q_stride, const void* k, const void* v,
                                         long long k_stride, long long v_stride, int pages, int page_rows,
                                         const void* table, long long table_stride, const void* lengths,
                                         const void* starts, int B, int W, int T, int qh, int kh, int d, float scale,
                                         void* out, void* workspace, long long workspace_bytes, int dtype, void* stream) {
    const PagedCache c = paged_cache(k, v, k_stride, v_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, (const int*)starts, B, W, table_stride};
    return prompt<Stage16>(q, q_stride, c, bt, T, qh, d, scale, out, workspace, workspace_bytes, dtype, stream);
}

MOSS_API int moss_paged_prompt_attention_fp8(const void* q, long long q_stride, const void* k, const void* v, const void* k_scales,
                                             const void* v_scales, long long k_stride, long long v_stride,
                                             long long k_scale_stride, long long v_scale_stride, int pages, int page_rows,
                                             const void* table, long long table_stride, const void* lengths,
                                             const void* starts, int B, int W, int T, int qh, int kh, int d, float scale,
                                             void* out, void* workspace, long long workspace_bytes, int dtype, void* stream) {
    const PagedCache8 c = paged_cache8(k, v, k_scales, v_scales, k_stride, v_stride, k_scale_stride, v_scale_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, (const int*)starts, B, W, table_stride};
    MOSS_CHECK_ARG(paged8_ok(c));
    return prompt<Stage8>(q, q_stride, c, bt, T, qh, d, scale, out, workspace, workspace_bytes, dtype, stream);
}
