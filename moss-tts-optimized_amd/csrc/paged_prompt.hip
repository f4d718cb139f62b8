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
// P's rounding is the one step with fewer bits before the output, as in the single request's prompt attention; the sum adds
// up the unrounded values.  (P = 2^(s scale - m) with m a rounded product: a row's largest P is 1 up to that rounding, which
// l and O share.)  Split into two 16-bit values as the decode form has it, P adds nothing to the output's own rounding, but
// costs half as many matrix instructions again where they are what bounds: 8000 tokens 555 -> 724 us, nine prompts 60 -> 67,
// for an error against 64 bits of 1.65 instead of 1.88 and 1.64 instead of 1.78 10^-3 (heads of 128, bf16; fp16 an eighth).
// Blocks of 64 keys go from the pages straight into LDS (buffer loads, 16 rows of K and of V a wave, which lie in one page;
// rows that nobody sees or that have no page are read as zeros: past the buffer's end), into one of two stages while the
// other is consumed: one barrier per block, no registers.  V is read transposed (ds_read_b64_tr_b16: a lane gets one
// dim of 4 rows).  16-byte chunk c of row r lies at c ^ f(r), which spreads the rows of one read over the banks.
// What bounds it: the matrix and vector pipes in turn at the clock that power holds (8000 tokens of 32 / 8 heads of 128:
// 520 to 550 us, 950 to 1010 TFLOP/s, where a large product of bf16 matrices reaches 1640); with K and V through registers, V
// transposed on the way, 667 us.
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

// A workgroup's sequence and its item's number, of what count(tiles, share) counts; `first`: partial results of the
// sequences taken before it.  A batch of up to 64 is one read of lengths and starts, and taken in the order of its lengths.
struct Found {
    PromptTiles tiles;
    int b, tok0, index, share, first;  // b -1: none
};
template <int HEIGHT, typename Count>
__device__ __forceinline__ Found find_tile(const PromptArgs& a, const PagedCache& c, const PagedBatch& bt, int item, int lane,
                                           Count count) {
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };  // it is; this puts it into a scalar
    auto of = [&](int b, int& tok0) {
        const int2 t = paged_tokens(bt, b, a.T);
        tok0 = t.x;
        return PromptTiles{t.y, a.group, paged_length(bt, b, c.shift) - t.y, HEIGHT};
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

template <typename E, int D, int KS>
__global__ __launch_bounds__(256, 2) void paged_prompt_kernel(PromptArgs a, PagedCache c, PagedBatch bt) {
    constexpr int RW = 4 / KS, NT = 2 / KS, HEIGHT = 32 * RW;  // row waves; a wave's 32-key tiles of a block
    constexpr int BK = kPromptBlock, DT = D / 32, DK = D / 16, RB = 2 * D;  // RB: bytes of a row
    constexpr int KB = BK * RB, NL = 16 * RB / 1024, RPL = 1024 / RB, CPR = D / 8;  // loads of 16 rows, rows of a load
    // two stages of K | V: two variables, so that reading one does not wait for the loads into the other
    __shared__ __attribute__((aligned(1024))) unsigned char even[2 * KB], odd[2 * KB];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, rl = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rw = wave % RW, kq = wave / RW;
    const int kvh = blockIdx.x % c.kh, G = a.group;  // neighbours in the grid, which lie on different XCDs, differ in it
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const Found f = find_tile<HEIGHT>(a, c, bt, (int)(blockIdx.x / c.kh), lane,
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
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;  // l: this lane's keys only

    // Blocks are taken from the last one down, so that the ones that not all rows see come first.
    // pages: lane i holds that of 16-row group i % 4 of the i / 4-th of the next 16 blocks (-1: none, or behind the last key);
    // bit i of `there` says that the group's rows up to the last key exist
    const int* trow = bt.table + (size_t)f.b * bt.table_stride;
    int pages = -1;
    unsigned long long there = 0, there_next = 0;
    auto fetch_pages = [&](int b) {
        const int key = BK * (b - lane / 4) + 16 * (lane & 3);
        pages = key >= 0 && key <= last ? page_or_none(trow[key >> c.shift], c.pages) : -1;
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
        if (((b1 - 1 - b) & 15) == 0) fetch_pages(b);
        const int page = __builtin_amdgcn_readlane(pages, 4 * ((b1 - 1 - b) & 15) + wave), key = BK * b + 16 * wave;
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
    for (int kk = 0; kk < DK; ++kk) kread[kk] = (uint32_t)((32 * kq + rl) * RB + 16 * ((2 * kk + half) ^ k_swizzle<D>(rl)));
    {
        const int i = lane & 15, r = 4 * half + (i >> 2), chunk = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                vread[s2][dt] = (uint32_t)((32 * kq + r + 8 * s2) * RB + 16 * ((4 * dt + chunk) ^ v_swizzle<D>(r + 8 * s2)) + 8 * (i & 1));
    }

    // O of this wave's keys from block b on, one key at a time and from memory, each row taking the keys it sees alone.
    auto again = [&](int b) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
        for (int j = 0; j < 32 * NT * (b1 - b); ++j) {
            const int key = uniform(BK * (b + j / (32 * NT)) + 32 * kq + j % (32 * NT));
            if (key > wave_last) break;
            const int page = uniform(page_of_row(trow, key, bt.W, c.shift, c.pages));
            if (page < 0) continue;
            const uint16_t* kp = c.k + row_offset(page, c.k_stride, kvh, key, c.shift, D) + 8 * half;
            const uint16_t* vp = c.v + row_offset(page, c.v_stride, kvh, key, c.shift, D) + 4 * half;
            float dot = 0.f;
#pragma unroll
            for (int kk = 0; kk < DK; ++kk) {
                const u32x4_t kw = *reinterpret_cast<const u32x4_t*>(kp + 16 * kk);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    dot = fmaf(E::hi(qf[kk][i]), E::hi(kw[i]), fmaf(E::lo(qf[kk][i]), E::lo(kw[i]), dot));
            }
            dot = sum_xor32(dot);
            if (key > qpos) continue;
            const float p = __builtin_amdgcn_exp2f(fmaf(dot, a.scale, -(m == -INFINITY ? 0.f : m)));
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const u32x2_v v = *reinterpret_cast<const u32x2_v*>(vp + 32 * dt + 8 * q4);
                    o[dt][4 * q4] = fmaf(p, E::lo(v[0]), o[dt][4 * q4]);
                    o[dt][4 * q4 + 1] = fmaf(p, E::hi(v[0]), o[dt][4 * q4 + 1]);
                    o[dt][4 * q4 + 2] = fmaf(p, E::lo(v[1]), o[dt][4 * q4 + 2]);
                    o[dt][4 * q4 + 3] = fmaf(p, E::hi(v[1]), o[dt][4 * q4 + 3]);
                }
        }
    };
    auto block = [&](const unsigned char* ks, unsigned char* next, int b) {
        // this wave's rows of block b are there, then everyone's; and everyone is done with block b + 1's stage
        __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // vmcnt(0)
        __syncthreads();
        if (((b1 - 1 - b) & 15) == 0) there = there_next;
        const int first = BK * b + 32 * kq;  // this wave's keys: 32 NT from here on, and their 16-row groups
        const unsigned int groups = (unsigned int)(there >> (4 * ((b1 - 1 - b) & 15) + 2 * kq)) & ((1u << 2 * NT) - 1);
        if (b > b0) copy(next, b - 1);
        if (idle || first > wave_last) return;  // none of its rows sees any of its keys
        const unsigned char* vs = ks + KB;
        f32x16_v s[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) s[i] = f32x16_v{};
#pragma unroll
        for (int kk = 0; kk < DK; ++kk)
#pragma unroll
            for (int i = 0; i < NT; ++i)
                s[i] = E::mfma32(*reinterpret_cast<const u32x4_t*>(ks + kread[kk] + 32 * RB * i), qf[kk], s[i]);
        // element e of tile i: key first + 32 i + 8 (e / 4) + 4 half + e % 4, row rl
        if (groups != (1u << 2 * NT) - 1 || first + 32 * NT - 1 > wave_first) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = first + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3);
                    s[i][e] = key <= qpos && (groups >> (2 * i + (e >> 3)) & 1) ? s[i][e] : -INFINITY;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 2) mx = fmaxf(fmaxf(mx, s[i][e]), s[i][e + 1]);
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
        for (int i = 0; i < NT; ++i) {
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
        if (first + 32 * NT - 1 > wave_first) {
            // A P of 0 times a NaN or infinity in V of a key that a row does not see is a NaN all the same.
            float z = 0.f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) z = fmaf(o[dt][e], 0.f, z);
            if (__any(z != z)) again(b);
        }
    };
    if (b0 < b1) copy(even, b1 - 1);
    for (int b = b1 - 1; b >= b0; b -= 2) {
        block(even, odd, b);
        if (b > b0) block(odd, even, b - 1);
    }
    l = sum_xor32(l);
    if constexpr (KS > 1) {
        // the second wave of the same rows hands over m, l and O in LDS; both scale to the larger m
        __syncthreads();
        float4* ox = reinterpret_cast<float4*>(rw ? odd : even);  // [dt][e / 4][lane], then m and l
        float* ml = reinterpret_cast<float*>(ox + DT * 4 * 64);
        if (kq == 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    ox[(4 * dt + j) * 64 + lane] = make_float4(o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]);
            ml[lane] = m;
            ml[64 + lane] = l;
        }
        __syncthreads();
        if (kq == 1) return;
        const float m1 = ml[lane], mn = fmaxf(m, m1);
        const float f0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        const float f1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - mn);
        m = mn;
        l = l * f0 + ml[64 + lane] * f1;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 v = ox[(4 * dt + j) * 64 + lane];
                o[dt][4 * j] = o[dt][4 * j] * f0 + v.x * f1;
                o[dt][4 * j + 1] = o[dt][4 * j + 1] * f0 + v.y * f1;
                o[dt][4 * j + 2] = o[dt][4 * j + 2] * f0 + v.z * f1;
                o[dt][4 * j + 3] = o[dt][4 * j + 3] * f0 + v.w * f1;
            }
    }
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
__global__ __launch_bounds__(2 * HEIGHT) void paged_prompt_join(PromptArgs a, PagedCache c, PagedBatch bt) {
    const int lane = threadIdx.x & 63, r = threadIdx.x % HEIGHT, h = threadIdx.x / HEIGHT, kvh = blockIdx.x % c.kh, G = a.group;
    const Found f = find_tile<HEIGHT>(a, c, bt, (int)(blockIdx.x / c.kh), lane,
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
        const size_t at = ((size_t)slot * c.kh + kvh) * HEIGHT + r;
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
// Parts of the whole call's work, over all KV heads, that a tile is not cut below.  128 / 256 / 512: 29 / 22 / 23 us for 150
// tokens after 1900, 61 / 46 / 47 for 32 single tokens after 50 to 4000, 46 / 46 / 49 for the nine prompts.
constexpr int kShares = 256;

PromptPlan prompt_plan(int B, int W, int shift, int T, int qh, int kh) {
    PromptPlan p;
    const long long rows = (long long)T * (qh / kh);
    p.height = (rows + 127) / 128 * kh <= kSmallTiles ? 64 : 128;
    p.tiles = (rows + p.height - 1) / p.height + (B < T ? B : T);
    p.shares = kShares / kh > 1 ? kShares / kh : 1;
    const long long parts = (((long long)W << shift) + kPromptShare * kPromptBlock - 1) / (kPromptShare * kPromptBlock);
    p.slots = parts <= 1 ? 0 : p.tiles * parts < 2 * p.shares ? p.tiles * parts : 2 * p.shares;
    return p;
}

template <typename E, int D, int KS>
int launch_prompt(const PromptArgs& a, const PagedCache& c, const PagedBatch& bt, const PromptPlan& p, hipStream_t st) {
    constexpr int HEIGHT = 128 / KS;
    const long long groups = (p.tiles + (p.slots ? p.shares : 0)) * c.kh;
    MOSS_CHECK_ARG(groups * 256 < (1ll << 32));
    hipLaunchKernelGGL((paged_prompt_kernel<E, D, KS>), dim3((unsigned)groups), dim3(256), 0, st, a, c, bt);
    if (p.slots) {
        const long long cut = (p.tiles < p.shares ? p.tiles : p.shares) * c.kh;
        hipLaunchKernelGGL((paged_prompt_join<E, D, HEIGHT>), dim3((unsigned)cut), dim3(2 * HEIGHT), 0, st, a, c, bt);
    }
    return moss_launch_status();
}

template <typename E, int D>
int launch_prompt(const PromptArgs& a, const PagedCache& c, const PagedBatch& bt, const PromptPlan& p, hipStream_t st) {
    return p.height == 64 ? launch_prompt<E, D, 2>(a, c, bt, p, st) : launch_prompt<E, D, 1>(a, c, bt, p, st);
}

}  // namespace
}  // namespace moss

using namespace moss;

MOSS_API long long moss_paged_prompt_workspace_bytes(int B, int W, int page_rows, int T, int qh, int kh, int d) {
    const int shift = page_shift(page_rows);
    if (B <= 0 || W <= 0 || shift < 0 || ((long long)W << shift) > (1ll << 30) || T <= 0 || kh <= 0 || qh <= 0 || qh % kh ||
        (d != 64 && d != 128))
        return 0;
    const PromptPlan p = prompt_plan(B, W, shift, T, qh, kh);
    return p.slots * kh * p.height * (d + 2) * 4;
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
    const long long values = p.slots * kh * p.height;
    MOSS_CHECK_ARG(p.slots == 0 || (workspace && workspace_bytes >= values * (d + 2) * 4));
    const PromptArgs a{(const uint16_t*)q, q_stride, (uint16_t*)out, (float*)workspace,
                       reinterpret_cast<float2*>((float*)workspace + values * d), T, qh, qh / kh, p.shares,
                       p.slots, fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f), scale < 0.f ? 0x80008000u : 0u};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0)
        return d == 128 ? launch_prompt<Bf16, 128>(a, c, bt, p, st) : launch_prompt<Bf16, 64>(a, c, bt, p, st);
    return d == 128 ? launch_prompt<F16, 128>(a, c, bt, p, st) : launch_prompt<F16, 64>(a, c, bt, p, st);
}
