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
//   S^T = K Q^T: 32 keys x 32 rows per matrix instruction, so a lane holds one row and 16 of its keys, and the row's
//   maximum needs one exchange with the lane 32 away; the running maximum and sum are fp32, base 2.
//   O^T += V^T P^T: P, rounded to 16 bits, is the B operand as S^T left it.
// P's rounding is the one step with fewer bits before the output: the largest P of a block is exactly 1 or its
// share of the running maximum, and the sum adds up the unrounded values.
// Blocks of 64 keys go from the pages straight into LDS (buffer loads, 16 rows of K and of V a wave, which lie in one page;
// rows that nobody sees or that have no page are read as zeros: past the buffer's end), into one of two stages while the
// other is consumed: one barrier per block, no registers.  V is read transposed (ds_read_b64_tr_b16: a lane gets one
// dim of 4 rows).  16-byte chunk c of row r lies at c ^ f(r), which spreads the rows of one read over the banks.
#include "paged.h"

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

__device__ __forceinline__ PromptTiles prompt_tiles(const PagedBatch& bt, int b, int T, int group, int shift) {
    const int n = paged_tokens(bt, b, T).y;
    return PromptTiles{n, group, paged_length(bt, b, shift) - n};
}

// Blocks in a part: from all sequences' tiles, over the KV head's fair shares.
__device__ __forceinline__ int prompt_share_of(const PagedBatch& bt, int T, int group, int shift, int shares, int lane) {
    long long blocks = 0;
    for (int b = lane; b < bt.B; b += kWave) blocks += prompt_tiles(bt, b, T, group, shift).blocks_bound();
    return __builtin_amdgcn_readfirstlane(prompt_share(wave_total(blocks), shares));
}

// Partial results of the sequences before b.
__device__ __forceinline__ int parts_before(const PagedBatch& bt, int b, int T, int group, int shift, int share, int lane) {
    int n = 0;
    for (int s = lane; s < b; s += kWave) {
        const PromptTiles t = prompt_tiles(bt, s, T, group, shift);
        if (t.tiles_over(share)) n += t.parts(share);
    }
    return wave_total(n);
}

// Where 16-byte chunk c of key row r lies in its LDS row: c ^ f(r).
template <int D>
__device__ __forceinline__ int k_swizzle(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
template <int D>
__device__ __forceinline__ int v_swizzle(int r) {
    return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r >> 1 & 1) << 2) | ((r >> 2) & 3);
}

// 16 bytes per lane straight to lds + 16 lane.  (In a function of its own: the host's pass drops a kernel that names a
// builtin it does not know.)
__device__ __forceinline__ void copy16(const Span& s, unsigned char* lds, uint32_t voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(span_rsrc(s), lds, 16, voff, 0, 0, 0);
}

typedef short s16x4_v __attribute__((ext_vector_type(4)));
// 4 rows of one dim: a 16-lane group reads 4 rows of 16 dims, lane i the 8 bytes of row i / 4 from dim 4 (i % 4) on.
__device__ __forceinline__ u32x2_v read_transposed(const unsigned char* p) {
    return __builtin_bit_cast(u32x2_v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_v*)p));
}

template <typename E, int D>
__global__ __launch_bounds__(256, 2) void paged_prompt_kernel(PromptArgs a, PagedCache c, PagedBatch bt) {
    constexpr int BK = kPromptBlock, DT = D / 32, DK = D / 16, RB = 2 * D;  // RB: bytes of a row
    constexpr int KB = BK * RB, NL = 16 * RB / 1024, RPL = 1024 / RB, CPR = D / 8;  // loads of 16 rows, rows of a load
    // two stages of K | V: two variables, so that reading one does not wait for the loads into the other
    __shared__ __attribute__((aligned(1024))) unsigned char even[2 * KB], odd[2 * KB];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, rl = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % c.kh, G = a.group;  // neighbours in the grid, which lie on different XCDs, differ in it
    const int share = prompt_share_of(bt, a.T, G, c.shift, a.shares, lane);
    const Place pl = find_item(bt.B, (int)(blockIdx.x / c.kh), lane,
                               [&](int b) { return prompt_tiles(bt, b, a.T, G, c.shift).items(share); });
    if (pl.b < 0) return;
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };  // it is; this puts it into a scalar
    const int sequence = uniform(pl.b), tok0 = uniform(paged_tokens(bt, sequence, a.T).x);
    const PromptTiles all = prompt_tiles(bt, sequence, a.T, G, c.shift);
    const PromptTiles tiles{uniform(all.tokens), G, uniform(all.pos0)};
    const PromptItem found = prompt_item(tiles, share, uniform(pl.index));
    const PromptItem item{uniform(found.tile), uniform(found.part), uniform(found.slot)};
    const int pos0 = tiles.pos0;
    const int row0 = item.tile * kPromptRows, nrows = tiles.rows();
    const int row = min(row0 + 32 * wave + rl, nrows - 1);  // this lane's row (clamped: stores are guarded)
    const int token = row / G, head = kvh * G + row % G;
    const int qpos = pos0 + token;  // sees keys 0 .. qpos
    const int last = uniform(tiles.last_key(item.tile)), blocks = uniform(tiles.blocks(item.tile));  // the workgroup's last key
    const bool cut = blocks > share, idle = row0 + 32 * wave >= nrows;             // idle: no row of this wave's exists
    const int wave_last = uniform(pos0 + min(row0 + 32 * wave + 31, nrows - 1) / G);
    const int wave_first = uniform(pos0 + min(row0 + 32 * wave, nrows - 1) / G);  // keys up to it are seen by all its rows
    const int b0 = uniform(item.part * share), b1 = uniform(min(blocks, b0 + share));

    u32x4_t qf[DK];  // lane: row rl, dims 16 kk + 8 half .. + 7
    {
        const uint16_t* qr = a.q + (size_t)(tok0 + token) * a.q_stride + (size_t)head * D + 8 * half;
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) qf[kk] = *reinterpret_cast<const u32x4_t*>(qr + 16 * kk) ^ a.flip;
    }
    f32x16_v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;  // l: this lane's keys only

    // pages: lane i holds that of 16-row group i of 16 blocks (-1: none, or behind the last key); bit i of `there` says
    // that the group's rows up to the last key exist
    const int* trow = bt.table + (size_t)sequence * bt.table_stride;
    int pages = -1;
    unsigned long long there = 0, there_next = 0;
    auto fetch_pages = [&](int b) {
        const int key = BK * b + 16 * lane;
        pages = key <= last ? page_or_none(trow[key >> c.shift], c.pages) : -1;
        there_next = __ballot(pages >= 0 || key > last);
    };
    // LDS offsets: this lane's part of a load, and what it reads
    uint32_t kload[NL], vload[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        const int r = j * RPL + lane / CPR, slot = lane % CPR;
        kload[j] = (uint32_t)(r * RB + 16 * (slot ^ k_swizzle<D>(r)));
        vload[j] = (uint32_t)(r * RB + 16 * (slot ^ v_swizzle<D>(r)));
    }
    auto copy = [&](unsigned char* stage, int b) {  // block b's rows 16 wave .. + 15
        if (((b - b0) & 15) == 0) fetch_pages(b);
        const int page = __builtin_amdgcn_readlane(pages, 4 * ((b - b0) & 15) + wave), key = BK * b + 16 * wave;
        const uint32_t bytes = (uint32_t)uniform(page < 0 ? 0 : min(max(last + 1 - key, 0), 16) * RB);
        const Span ks{c.k + row_offset(page, c.k_stride, kvh, key, c.shift, D), bytes};
        const Span vs{c.v + row_offset(page, c.v_stride, kvh, key, c.shift, D), bytes};
        unsigned char* at = stage + 16 * RB * wave;
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            copy16(ks, at + 1024 * j, kload[j]);
            copy16(vs, at + KB + 1024 * j, vload[j]);
        }
    };
    uint32_t kread[DK], vread[2][DT];
#pragma unroll
    for (int kk = 0; kk < DK; ++kk) kread[kk] = (uint32_t)(rl * RB + 16 * ((2 * kk + half) ^ k_swizzle<D>(rl)));
    {
        const int i = lane & 15, r = 4 * half + (i >> 2), chunk = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                vread[s2][dt] = (uint32_t)((r + 8 * s2) * RB + 16 * ((4 * dt + chunk) ^ v_swizzle<D>(r + 8 * s2)) + 8 * (i & 1));
    }

    auto block = [&](const unsigned char* ks, unsigned char* next, int b) {
        // this wave's rows of block b are there, then everyone's; and everyone is done with block b - 1's stage
        __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // vmcnt(0)
        __syncthreads();
        if (((b - b0) & 15) == 0) there = there_next;
        const unsigned int groups = (unsigned int)(there >> (4 * ((b - b0) & 15))) & 15u;
        if (b + 1 < b1) copy(next, b + 1);
        if (idle || BK * b > wave_last) return;  // none of its rows sees any of its keys
        const unsigned char* vs = ks + KB;
        f32x16_v s[2];
        s[0] = f32x16_v{};
        s[1] = f32x16_v{};
#pragma unroll
        for (int kk = 0; kk < DK; ++kk)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                s[i] = E::mfma32(*reinterpret_cast<const u32x4_t*>(ks + kread[kk] + 32 * RB * i), qf[kk], s[i]);
        // element e of tile i: key BK b + 32 i + 8 (e / 4) + 4 half + e % 4, row rl
        if (groups != 15u || BK * b + BK - 1 > wave_first) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = BK * b + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3);
                    s[i][e] = key <= qpos && (groups >> (2 * i + (e >> 3)) & 1) ? s[i][e] : -INFINITY;
                }
        }
        float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(fmaxf(mx, s[0][e]), s[1][e]);
        mx = max_xor32(mx) * a.scale;
        if (__any(mx > m)) {
            const float mn = fmaxf(m, mx);
            const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= f;
        }
        const float mr = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u32x4_t pf[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[i][8 * u + 2 * v], a.scale, -mr));
                    const float p1 = __builtin_amdgcn_exp2f(fmaf(s[i][8 * u + 2 * v + 1], a.scale, -mr));
                    l += p0 + p1;
                    pf[u][v] = E::pack(p0, p1);
                }
            // K step u: keys 16 u + {4 half + 0..3, 8 + 4 half + 0..3} of the tile
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const u32x2_v a0 = read_transposed(vs + vread[0][dt] + (32 * i + 16 * u) * RB);
                    const u32x2_v a1 = read_transposed(vs + vread[1][dt] + (32 * i + 16 * u) * RB);
                    o[dt] = E::mfma32(u32x4_t{a0[0], a0[1], a1[0], a1[1]}, pf[u], o[dt]);
                }
        }
    };
    if (b0 < b1) copy(even, b0);
    for (int b = b0; b < b1; b += 2) {
        block(even, odd, b);
        if (b + 1 < b1) block(odd, even, b + 1);
    }
    l = sum_xor32(l);
    // O^T element e of d tile dt: d = 32 dt + 8 (e / 4) + 4 half + e % 4
    if (cut) {
        const int before = parts_before(bt, sequence, a.T, G, c.shift, share, lane);
        // (starts that do not rise can name more parts than there are tokens for: they have no slot)
        if (row0 + 32 * wave + rl >= nrows || before + item.slot >= a.slots) return;
        const size_t at = (size_t)(before + item.slot) * c.kh + kvh;
        float4* part = reinterpret_cast<float4*>(a.part) + at * (D / 4) * kPromptRows + 32 * wave + rl;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                part[(8 * dt + 2 * q4 + half) * kPromptRows] =
                    make_float4(o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]);
        if (half == 0) a.stat[at * kPromptRows + 32 * wave + rl] = make_float2(m, l);
        return;
    }
    if (row0 + 32 * wave + rl >= nrows) return;
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

// The parts of one cut tile and KV head, 256 threads: thread (row, h) takes the 4-dim pieces h, h + 2, .. of the row.
template <typename E, int D>
__global__ __launch_bounds__(256) void paged_prompt_join(PromptArgs a, PagedCache c, PagedBatch bt) {
    const int lane = threadIdx.x & 63, r = threadIdx.x & 127, h = threadIdx.x >> 7, kvh = blockIdx.x % c.kh, G = a.group;
    const int share = prompt_share_of(bt, a.T, G, c.shift, a.shares, lane);
    const Place pl = find_item(bt.B, (int)(blockIdx.x / c.kh), lane,
                               [&](int b) { return prompt_tiles(bt, b, a.T, G, c.shift).tiles_over(share); });
    if (pl.b < 0) return;
    const PromptTiles tiles = prompt_tiles(bt, pl.b, a.T, G, c.shift);
    const int tile = tiles.tiles() - 1 - pl.index, row = tile * kPromptRows + r;
    const int count = (tiles.blocks(tile) + share - 1) / share;
    const int before = parts_before(bt, pl.b, a.T, G, c.shift, share, lane);
    // part k's slot: the cut tiles' parts 0, then the tiles' of more than k shares
    auto number_of = [&](int k) {
        int slot = before + pl.index;
        for (int i = 0; i < k; ++i) slot += tiles.tiles_over(i ? i * share : share);
        return slot;
    };
    auto slot_of = [&](int k) { return ((size_t)number_of(k) * c.kh + kvh) * kPromptRows; };
    if (row >= tiles.rows() || number_of(count - 1) >= a.slots) return;
    float mx = -INFINITY, den = 0.f;
    for (int k = 0; k < count; ++k) mx = fmaxf(mx, a.stat[slot_of(k) + r].x);
    float4 acc[D / 8];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < count; ++k) {
        const size_t at = slot_of(k);
        const float2 st = a.stat[at + r];
        const float f = st.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.x - mx);
        den = fmaf(f, st.y, den);
        const float4* part = reinterpret_cast<const float4*>(a.part) + at * (D / 4) + r;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const float4 v = part[(2 * i + h) * kPromptRows];
            acc[i].x = fmaf(f, v.x, acc[i].x);
            acc[i].y = fmaf(f, v.y, acc[i].y);
            acc[i].z = fmaf(f, v.z, acc[i].z);
            acc[i].w = fmaf(f, v.w, acc[i].w);
        }
    }
    const float inv = den == 0.f ? 0.f : 1.0f / den;
    uint16_t* dst = a.out + ((size_t)(paged_tokens(bt, pl.b, a.T).x + row / G) * a.qh + kvh * G + row % G) * D;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<uint2*>(dst + 4 * (2 * i + h)) =
            make_uint2(E::pack(acc[i].x * inv, acc[i].y * inv), E::pack(acc[i].z * inv, acc[i].w * inv));
}

// Tiles at most, shares of a KV head, partial results at most (0: no tile can see more than a share's least blocks).
struct PromptPlan {
    long long tiles, slots;
    int shares;
};
constexpr int kShares = 512;  // workgroups of all KV heads that the work is shared out over: two a CU

PromptPlan prompt_plan(int B, int W, int shift, int T, int qh, int kh) {
    PromptPlan p;
    p.tiles = ((long long)T * (qh / kh) + kPromptRows - 1) / kPromptRows + (B < T ? B : T);
    p.shares = kShares / kh > 1 ? kShares / kh : 1;
    const long long parts = (((long long)W << shift) + kPromptShare * kPromptBlock - 1) / (kPromptShare * kPromptBlock);
    p.slots = parts <= 1 ? 0 : p.tiles * parts < 2 * p.shares ? p.tiles * parts : 2 * p.shares;
    return p;
}

template <typename E, int D>
int launch_prompt(const PromptArgs& a, const PagedCache& c, const PagedBatch& bt, const PromptPlan& p, hipStream_t st) {
    const long long groups = (p.tiles + (p.slots ? p.shares : 0)) * c.kh;
    MOSS_CHECK_ARG(groups * 256 < (1ll << 32));
    hipLaunchKernelGGL((paged_prompt_kernel<E, D>), dim3((unsigned)groups), dim3(256), 0, st, a, c, bt);
    if (p.slots) {
        const long long cut = (p.tiles < p.shares ? p.tiles : p.shares) * c.kh;
        hipLaunchKernelGGL((paged_prompt_join<E, D>), dim3((unsigned)cut), dim3(256), 0, st, a, c, bt);
    }
    return moss_launch_status();
}

}  // namespace
}  // namespace moss

using namespace moss;

MOSS_API long long moss_paged_prompt_workspace_bytes(int B, int W, int page_rows, int T, int qh, int kh, int d) {
    const int shift = page_shift(page_rows);
    if (B <= 0 || W <= 0 || shift < 0 || ((long long)W << shift) > (1ll << 30) || T <= 0 || kh <= 0 || qh <= 0 || qh % kh ||
        (d != 64 && d != 128))
        return 0;
    return prompt_plan(B, W, shift, T, qh, kh).slots * kh * kPromptRows * (d + 2) * 4;
}

MOSS_API int moss_paged_prompt_attention(const void* q, long long q_stride, const void* k, const void* v,
                                         long long k_stride, long long v_stride, int pages, int page_rows,
                                         const void* table, long long table_stride, const void* lengths,
                                         const void* starts, int B, int W, int T, int qh, int kh, int d, float scale,
                                         void* out, void* workspace, long long workspace_bytes, int dtype, void* stream) {
    const PagedCache c = paged_cache(k, v, k_stride, v_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, (const int*)starts, B, W, table_stride};
    MOSS_CHECK_ARG(q && out && starts && paged_pointers_ok(c, bt) && paged_shape_ok(c, bt, qh, d));
    MOSS_CHECK_ARG((dtype == 0 || dtype == 1) && T > 0 && T <= (1 << 20) && q_stride % 8 == 0 &&
                   q_stride >= (long long)qh * d && scale == scale);
    MOSS_CHECK_ARG(MOSS_ALIGNED(q, 16) && MOSS_ALIGNED(out, 16) && MOSS_ALIGNED(workspace, 16));
    const PromptPlan p = prompt_plan(B, W, c.shift, T, qh, kh);
    const long long values = p.slots * kh * kPromptRows;
    MOSS_CHECK_ARG(p.slots == 0 || (workspace && workspace_bytes >= values * (d + 2) * 4));
    const PromptArgs a{(const uint16_t*)q, q_stride, (uint16_t*)out, (float*)workspace,
                       reinterpret_cast<float2*>((float*)workspace + values * d), T, qh, qh / kh, p.shares,
                       p.slots, fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f), scale < 0.f ? 0x80008000u : 0u};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0)
        return d == 128 ? launch_prompt<Bf16, 128>(a, c, bt, p, st) : launch_prompt<Bf16, 64>(a, c, bt, p, st);
    return d == 128 ? launch_prompt<F16, 128>(a, c, bt, p, st) : launch_prompt<F16, 64>(a, c, bt, p, st);
}
