// Attention of one new token per sequence over a paged cache, where sequences that stand next to each other in the batch share the
// first rows of their caches: those are read and multiplied once for all of them.
//
// o_h = sum_t softmax_t(scale q_h . k_t) v_t over the rows t < length, as paged_decode.hip has it.  A run is neighbouring
// sequences with the same group number (not below 0); runs end at every 64th sequence of the batch, so a wave sees
// whole ones.  Of the rows that a run's first sequence shares (at most its length, whole 16 rows), sequence b takes the first n_b =
// shared[b], whole 16 rows, or all of its length if that is no more, from the pages of the first one, and the rest
// from its own.  P is what the others take at most, which the first one then takes too.  A run of one shares nothing.
//
// The prefix: all of a run's query heads of a KV head are the rows of tiles, which go over the keys on the matrix cores
// (paged_prompt.h), row b up to key n_b.  The rest: paged_decode.h, from row n_b on.  Both split P into two 16-bit values, so that
// what a sequence gets is as near to the definition whoever stands beside it; both leave (m, l, O), and a last launch
// joins a sequence's.
//
// Who takes what follows from groups, shared and lengths on the device, so that a captured graph follows them.  The work of a KV
// head are two lines: the blocks of 64 keys of every tile, tile after tile, and the units of 64 own rows of every sequence.
// Of the workgroups (two a CU in all), some take the first, a piece each, and the others the second, a piece a wave, in the
// proportion of what the lines cost; a piece that passes the end of a tile or a sequence leaves more than one result.  The
// last workgroup also writes where the join finds a sequence's parts.
//
// What bounds it: 64 sequences of 30 to 1500 own rows over 4096 shared ones (32 / 8 heads of 128, bf16) 35 us (decode_attention
// 102): the own rows, 92 of the 110 MB that it reads, come by single waves with one tile on its way each, four a CU beside a
// workgroup of the prefix's; parts are 11.6 MB, written and read again by the join (5 us).  With a launch each for prefix and rest
// it took 59, with the shares of a sequence as workgroups 50, own rows by whole workgroups 41.  40 in five runs over an 8-bit cache
// 26.9 us; four over 640 rows, which are not worth sharing, 10.9; sequences that share nothing about as decode_attention does (64
// of 4 to 8 thousand rows 256 for 273, from 8 bits 148 for 158; 16 of 17 to 8000 rows 20 for 18, from 8 bits 17 for 14).  More than
// 64 sequences, which every workgroup looks through 64 at a time: 128 over 4096 shared rows 47 us (decode_attention 190), 256 125
// (429).
// Registers: the instances for heads of 128 spill 2 / 16 (16 bits, tiles of 64 / 128 rows) or 18 / 34 (8 bits); those for heads of 64
// none, and of them only the one for 16 bits (bf16) and tiles of 64 rows has three waves a SIMD.
#include "paged_decode.h"
#include "paged_prompt.h"

namespace moss {
namespace {

// Over all KV heads: as many as there are places for.  448 / 512 / 768: 39.8 / 37.8 / 49.9 us for 64 sequences over 4096 shared rows
// (in a graph over three caches in turn).
constexpr int kWorkgroups = 512;

// Rows of a KV head that sharing has to save in a batch, over all KV heads.  Every sequence alone / shared, us, in this kernel: 8
// sequences over 640 shared rows of 32 / 8 heads (35840) 13.9 / 15.4, 32 over 256 (63488) 18.8 / 18.6, 16 over 640 (76800) 18.0 /
// 17.1, 4 over 4096 (98304) 21.6 / 21.0, 8 over 4096 (229376) 26 / 20; 16 / 1 heads, 16 over 4096 (61440) 25.5 / 28.3, 32 over
// 4096 (126976) 31.7 / 26.2; 12 / 12 heads of 64, 8 over 640 (53760) 13.6 / 14.1, 16 over 640 (115200) 16.4 / 14.9.  What the
// shared rows cost alone is so little because the caches serve all but the first reader.  Those were small caches; from pools past
// kCached, up to 40 in turn, with 50 own rows each: 32 / 8 heads, 8 over 640 12.4 / 13.8, 32 over 256 16.5 / 14.1, 16 over 640 17.3 /
// 17.1, 4 over 4096 22.8 / 18.9, 8 over 4096 35 / 19; 16 / 1 heads, 16 over 4096 24.0 / 21.1; from 8 bits 16 over 640 15.5 / 16.0,
// 4 over 4096 18.4 / 17.2, 8 over 4096 23.6 / 17.8.
constexpr int kWorth = 65536;

struct SharedArgs {
    DecodeArgs a;             // part and stat: of the sequences' own rows
    const int* groups;        // [B]
    const int* shared;        // [B]
    float* prefix_part;       // [KH, rows, D]
    float2* prefix_stat;      // [KH, rows]
    long long prefix_rows;
    struct Found* found;      // [B]
    int worth;                   // rows in sixteens that have to be saved
    int workgroups, head_tiles;  // workgroups of a KV head; tiles of 16 of its heads, for the own rows
};

// Sequence b0 + lane of the batch: where its own rows begin, and its run.
struct Member {
    int length, from;  // its rows, of which the first `from` are the run's
    int first, size;   // the run's lanes
    int rows;          // P; 0 for a run of one or of which nobody else takes any
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
    const int rows = m.size > 1 ? shared_rows(__shfl(want, m.first), __shfl(m.length, m.first)) : 0;
    // what those behind the first one take of them: the largest over the run, whose first lane stands above the value, in sixteens
    const int taken = taken_rows(m.first == lane ? 0 : shared_from(rows, want, m.length)) >> 4;
    const uint32_t most = wave_prefix_max((uint32_t)m.first << 26 | (uint32_t)min(taken, (1 << 26) - 1));
    m.rows = (int)(__shfl(most, m.first + m.size - 1) & ((1u << 26) - 1)) << 4;
    m.from = shared_from(m.rows, want, m.length);
    return m;
}

// Whether sharing saves enough rows to be worth the prefix's own way; if not, every sequence is taken alone.  (Rows in sixteens,
// and no more of a sequence than decide by themselves, so that the sum fits 32 bits.)  What is saved is what every sequence but
// one takes of the prefix: the first takes all that is read.
__device__ __forceinline__ int saved_by(const Member& m, int lane) {
    return m.first == lane ? 0 : min(m.from >> 4, 1 << 14);
}
template <typename At>
__device__ __forceinline__ bool worth_sharing(const SharedArgs& s, int B, int lane, At at) {
    if (B <= kWave) return wave_total(saved_by(at(0), lane)) >= s.worth;
    for (int b0 = 0, saved = 0; b0 < B; b0 += kWave) {
        saved += wave_total(saved_by(at(b0), lane));  // ends at the first that is enough: no overflow
        if (saved >= s.worth) return true;
    }
    return false;
}
// Members as they are taken.
struct Members {
    const SharedArgs& s;
    const PagedBatch& bt;
    int shift, lane;
    Member m0;
    bool worth;
    __device__ __forceinline__ Members(const SharedArgs& s, const PagedBatch& bt, int shift, int lane)
        : s(s), bt(bt), shift(shift), lane(lane), m0(member_of(s, bt, shift, 0, lane)) {
        worth = worth_sharing(s, bt.B, lane, [&](int b0) { return b0 == 0 ? m0 : member_of(s, bt, shift, b0, lane); });
        if (!worth) m0.from = m0.rows = 0;
    }
    __device__ __forceinline__ Member operator()(int b0) const {
        if (b0 == 0) return m0;
        Member m = member_of(s, bt, shift, b0, lane);
        if (!worth) m.from = m.rows = 0;
        return m;
    }
};

__device__ __forceinline__ long long shfl64(long long v, int lane) {
    return (long long)((unsigned long long)(unsigned)__shfl((int)(v >> 32), lane) << 32 | (unsigned)__shfl((int)v, lane));
}

// A run's tiles of `height` rows (of its first lane; 0 elsewhere), and their blocks of keys.
__device__ __forceinline__ int tiles_of(const Member& m, int group, int height, int lane) {
    return m.first == lane && m.rows > 0 ? (m.size * group + height - 1) / height : 0;
}
__device__ __forceinline__ int blocks_of(const Member& m) { return (m.rows + kPromptBlock - 1) / kPromptBlock; }

// The two lines of a KV head's work, how many workgroups take the first, and the pieces' lengths.  `at(b0)` gives the members from
// sequence b0 on.
struct Lines {
    long long blocks, units;
    int takers, blocks_each, units_each;
};
template <int HEIGHT, typename At>
__device__ __forceinline__ Lines lines_of(const SharedArgs& s, int B, int lane, At at) {
    long long blocks = 0, units = 0;
    for (int b0 = 0; b0 < B; b0 += kWave) {
        const Member m = at(b0);
        blocks += (long long)tiles_of(m, s.a.group, HEIGHT, lane) * blocks_of(m);
        units += own_units(m.own());
    }
    Lines l;
    l.blocks = wave_total(blocks), l.units = wave_total(units) * s.head_tiles;
    l.takers = __builtin_amdgcn_readfirstlane(prefix_takers((float)l.blocks, (float)l.units, s.workgroups));
    l.blocks_each = piece_of(l.blocks, max(l.takers, 1));
    l.units_each = piece_of(l.units, 4 * max(s.workgroups - l.takers, 1));
    return l;
}

// Where the tiles of the runs that begin at sequences b0 + lane lie.
struct Places {
    long long end;  // on the line of blocks; the lane's tiles lie before it
    int rows_end;   // rows of the tiles so far
    int tiles, blocks;
};
template <int HEIGHT>
__device__ __forceinline__ Places places_of(const SharedArgs& s, const Member& m, int lane, long long before, int rows_before) {
    Places p;
    p.tiles = tiles_of(m, s.a.group, HEIGHT, lane), p.blocks = p.tiles ? blocks_of(m) : 0;
    p.end = before + wave_prefix((long long)p.tiles * p.blocks);
    p.rows_end = rows_before + wave_prefix(p.tiles ? m.size * s.a.group : 0);
    return p;
}
// Where the own rows of sequences b0 + lane end on the line of units.
__device__ __forceinline__ long long units_end(const SharedArgs& s, const Member& m, long long before) {
    return before + wave_prefix((long long)own_units(m.own()) * s.head_tiles);
}

// What the join has to know of a sequence, written by the last workgroup: its run's first block on the line, the blocks of a
// tile (0: nothing shared), its row among the run's and among all partial rows; its first unit and units; the pieces.
struct Found {
    long long block, unit;
    int blocks, in_run, row, units;
    int blocks_each, units_each;
};

// The chunk of 64 sequences that a workgroup is at, in LDS: in registers it would lie beside the products' (50 of which went to
// memory).
struct Chunk {
    long long end[kWave];
    int rows_end[kWave], tiles[kWave], blocks[kWave];
    int from[kWave], size[kWave], rows[kWave];
    __device__ __forceinline__ void put(const Member& m, const Places& p, int lane) {  // by one wave
        end[lane] = p.end, rows_end[lane] = p.rows_end, tiles[lane] = p.tiles, blocks[lane] = p.blocks;
        from[lane] = m.from, size[lane] = m.size, rows[lane] = m.rows;
    }
};
// A value that is the same in all lanes, in a scalar.
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long long scalar(long long v) { return lane_value(v, 0); }

// Some blocks of a tile.
template <typename E, int D, int KS, typename S>
__device__ __forceinline__ void prefix_part(const SharedArgs& s, const typename S::Cache& c, const PagedBatch& bt, const Chunk& ch, int b0,
                                            int l, int tile, int from, int to, long long out0, int kvh, Stage<D>& even, Stage<D>& odd) {
    constexpr int HEIGHT = 128 / KS, RW = 4 / KS, DT = D / 32, DK = D / 16;
    const DecodeArgs& a = s.a;
    const int tid = fresh_thread(), lane = tid & (kWave - 1), half = lane >> 5, rl = lane & 31, G = a.group;
    const int rw = scalar(tid >> 6) % RW;
    const int nrows = scalar(ch.size[l]) * G, row = min(tile * HEIGHT + 32 * rw + rl, nrows - 1);  // clamped: stores are guarded
    const int token = (int)((unsigned)row / (unsigned)G), head = kvh * G + row - token * G;
    TileRows rows;
    rows.qpos = ch.from[l + token] - 1;
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
    rows.kvh = kvh, rows.b0 = from, rows.b1 = to, rows.last = scalar(ch.rows[l]) - 1;
    rows.wave_first = scalar(least), rows.wave_last = scalar(most);
    rows.idle = tile * HEIGHT + 32 * rw >= nrows;
    f32x16_v o[DT];
    float mx, sum;
    if (!attend_rows<E, D, KS, true, S>(c, rows, bt.W, qf, a.scale, tid, even, odd, o, mx, sum)) return;
    const long long out = out0 + 32 * rw + rl;
    if (tile * HEIGHT + 32 * rw + rl >= nrows || out < 0 || out >= s.prefix_rows) return;
    const size_t at = (size_t)kvh * s.prefix_rows + out;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<float4*>(s.prefix_part + at * D + 32 * dt + 8 * q4 + 4 * half) =
                make_float4(o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]);
    if (half == 0) s.prefix_stat[at] = make_float2(mx, sum);
}

// Grid: workgroups of a KV head * KV heads; neighbours, which lie on different XCDs, differ in the KV head.
template <typename E, int D, int KS, typename S, typename T, bool NT>
__global__ __launch_bounds__(256, 2) void paged_shared_split(SharedArgs s, typename S::Cache c, PagedBatch bt) {
    constexpr int HEIGHT = 128 / KS;
    __shared__ __attribute__((aligned(1024))) Stage<D> even, odd;
    __shared__ Chunk ch;
    const DecodeArgs& a = s.a;
    const int lane = threadIdx.x & (kWave - 1), G = a.group, kvh = blockIdx.x % c.kh, w = blockIdx.x / c.kh;
    const Members at(s, bt, c.shift, lane);
    const Member m0 = at(0);
    const Lines lines = lines_of<HEIGHT>(s, bt.B, lane, at);
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x < kWave) {
        Member m = m0;
        Places p = places_of<HEIGHT>(s, m, lane, 0, 0);
        long long ends = units_end(s, m, 0);
        for (int b0 = 0;;) {
            Found f;
            f.blocks = m.from > 0 ? __shfl(p.blocks, m.first) : 0;
            f.block = shfl64(p.end, m.first) - (long long)__shfl(p.tiles, m.first) * __shfl(p.blocks, m.first);
            f.in_run = (lane - m.first) * G;
            f.row = __shfl(p.rows_end, m.first) - m.size * G + f.in_run;
            f.units = own_units(m.own());
            f.unit = ends - (long long)f.units * s.head_tiles;
            f.blocks_each = lines.blocks_each, f.units_each = lines.units_each;
            if (b0 + lane < bt.B) s.found[b0 + lane] = f;
            b0 += kWave;
            if (b0 >= bt.B) break;
            const long long before = lane_value(p.end, kWave - 1), units = lane_value(ends, kWave - 1);
            const int rows = lane_value(p.rows_end, kWave - 1);
            m = at(b0);
            p = places_of<HEIGHT>(s, m, lane, before, rows);
            ends = units_end(s, m, units);
        }
    }
    if (w < lines.takers) {
        long long pos = (long long)w * lines.blocks_each;
        const long long end = min(pos + lines.blocks_each, lines.blocks);
        if (pos >= end) return;
        const bool writer = threadIdx.x < kWave;
        {
            const Places p = places_of<HEIGHT>(s, m0, lane, 0, 0);
            if (writer) ch.put(m0, p, lane);
            __syncthreads();
        }
        for (int b0 = 0;;) {
            const unsigned long long past = __ballot(ch.end[lane] > pos);
            if (!past) {  // further on
                b0 += kWave;
                if (b0 >= bt.B) return;
                const Member m = at(b0);
                const Places p = places_of<HEIGHT>(s, m, lane, ch.end[kWave - 1], ch.rows_end[kWave - 1]);
                __syncthreads();
                if (writer) ch.put(m, p, lane);
                __syncthreads();
                continue;
            }
            const int l = __builtin_ctzll(past), blocks = scalar(ch.blocks[l]);
            const long long in = pos - (scalar(ch.end[l]) - (long long)scalar(ch.tiles[l]) * blocks);
            const int tile = scalar((int)quotient(in, blocks)), from = scalar((int)(in - (long long)tile * blocks));
            const int to = scalar((int)min((long long)blocks, from + (end - pos)));
            const long long out = scalar(ch.rows_end[l]) - scalar(ch.size[l]) * G + tile * HEIGHT + (long long)w * HEIGHT;
            prefix_part<E, D, KS, S>(s, c, bt, ch, b0, l, tile, from, to, out, kvh, even, odd);
            pos += to - from;
            if (pos >= end) return;
            __syncthreads();  // everyone is done with the LDS
        }
    }
    const int v = (w - lines.takers) * 4 + scalar((int)threadIdx.x >> 6);
    long long pos = (long long)v * lines.units_each;
    const long long end = min(pos + lines.units_each, lines.units);
    if (pos >= end) return;
    Member m = m0;
    long long ends = units_end(s, m, 0);
    for (int b0 = 0; pos < end;) {
        const unsigned long long past = __ballot(ends > pos);
        if (!past) {
            b0 += kWave;
            if (b0 >= bt.B) return;
            m = at(b0);
            ends = units_end(s, m, lane_value(ends, kWave - 1));
            continue;
        }
        const int l = __builtin_ctzll(past), from = lane_value(m.from, l), rows = lane_value(m.length, l) - from, units = own_units(rows);
        const long long in = pos - (lane_value(ends, l) - (long long)units * s.head_tiles);
        const int tile = scalar((int)quotient(in, units)), u0 = scalar((int)(in - (long long)tile * units));
        const int u1 = scalar((int)min((long long)units, u0 + (end - pos)));
        pos += u1 - u0;
        ShareOf sh;
        sh.b = b0 + l, sh.slot = (long long)v + sh.b;
        sh.kvh = kvh, sh.h0 = 16 * tile, sh.heads = min(16, G - sh.h0);
        sh.r0 = from + u0 * kOwnUnit, sh.r1 = from + (int)min((long long)rows, (long long)u1 * kOwnUnit);
        sh.alone = from == 0 && u0 == 0 && u1 == units;
        if (sh.slot >= a.slots) return;
        float(&none)[2][4][16] = *reinterpret_cast<float(*)[2][4][16]>(odd);
        decode_share<E, D, T, NT, 1>(a, c, bt, sh, fresh_thread(), *reinterpret_cast<float(*)[4][16][D]>(even), none[0], none[1]);
    }
}

// grid (QH * WAVES / 4 rounded up, B), 256 threads: the parts of a head's prefix and of its sequence's own rows, by WAVES waves, wave w
// taking w, w + WAVES, .., whose sums meet in LDS.
template <typename E, int D, int HEIGHT, int WAVES>
__global__ __launch_bounds__(256) void paged_shared_join(SharedArgs s) {
    constexpr int VPL = D / kWave;
    const DecodeArgs& a = s.a;
    __shared__ float acc_s[4][D];
    const int lane = threadIdx.x & (kWave - 1), wave = scalar((int)threadIdx.x >> 6), w = wave % WAVES, b = blockIdx.y, G = a.group;
    const int h = blockIdx.x * (4 / WAVES) + wave / WAVES;
    if (h >= a.qh) return;  // (WAVES 4: never)
    const Found f = s.found[b];
    // the pieces that hold the tile's blocks, and those that hold the own rows
    int pieces = 0, pieces_own = 0, w0 = 0, w1 = 0;
    long long row = 0;
    if (f.blocks > 0) {
        const long long start = f.block + (long long)((f.in_run + h % G) / HEIGHT) * f.blocks;
        w0 = (int)quotient(start, f.blocks_each);
        pieces = (int)quotient(start + f.blocks - 1, f.blocks_each) - w0 + 1;
        row = f.row + h % G + (long long)w0 * HEIGHT;
    }
    if (f.units > 0) {
        const long long start = f.unit + (long long)f.units * (h % G / 16);
        w1 = (int)quotient(start, f.units_each);
        pieces_own = (int)quotient(start + f.units - 1, f.units_each) - w1 + 1;
    }
    if (pieces == 0 && pieces_own == 1) return;  // written by its workgroup
    const int count = pieces + pieces_own;
    const long long slot = (long long)w1 + b;
    if (pieces < 0 || pieces_own < 0 || slot < 0 || slot + pieces_own > a.slots || row < 0 ||
        (pieces && row + (long long)(pieces - 1) * HEIGHT >= s.prefix_rows))
        return;  // only where another call writes the same workspace
    // part i's place among the statistics and results: the prefix's, then the sequence's own
    const long long row0 = (long long)(h / G) * s.prefix_rows + row, row1 = slot * a.qh + h;
    auto stat = [&](int i) {
        return i < pieces ? s.prefix_stat[row0 + (long long)i * HEIGHT] : a.stat[row1 + (long long)(i - pieces) * a.qh];
    };
    auto part = [&](int i) {
        return (i < pieces ? s.prefix_part + (row0 + (long long)i * HEIGHT) * D : a.part + (row1 + (long long)(i - pieces) * a.qh) * D) +
               VPL * lane;
    };
    const float2 own = lane < count ? stat(lane) : make_float2(-INFINITY, 0.f);
    constexpr int N = WAVES == 4 ? 8 : 16;  // parts of a wave on their way together
    float x[N][VPL], acc[VPL], den = 0.f;
    auto load = [&](int i0) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float* from_part = part(min(i0 + WAVES * n, count - 1));
#pragma unroll
            for (int i = 0; i < VPL; ++i) x[n][i] = from_part[i];
        }
    };
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] = 0.f;
    if (count) {
        if (w < count) load(w);
        float mx = own.x;
        for (int i = kWave + lane; i < count; i += kWave) mx = fmaxf(mx, stat(i).x);
        mx = wave_max(mx);
        auto weight = [&](float v) { return v == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v - mx); };
        const float f0 = weight(own.x);
        den = f0 * own.y;
        for (int i = kWave + lane; i < count; i += kWave) {
            const float2 v = stat(i);
            den += weight(v.x) * v.y;
        }
        den = wave_sum(den);
        for (int i0 = w; i0 < count; i0 += WAVES * N) {
            if (i0 != w) load(i0);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int i = min(i0 + WAVES * n, count - 1);
                float f = i < kWave ? __uint_as_float(lane_value(__float_as_uint(f0), i)) : weight(stat(i).x);
                if (i0 + WAVES * n >= count) f = 0.f;
#pragma unroll
                for (int k = 0; k < VPL; ++k) acc[k] = f == 0.f ? acc[k] : fmaf(f, x[n][k], acc[k]);
            }
        }
    }
    const float inv = den == 0.f ? 0.f : 1.0f / den;
    uint16_t* dst = a.out + ((size_t)b * a.qh + h) * D;
    if constexpr (WAVES == 1) {
        if constexpr (VPL == 2)
            reinterpret_cast<uint32_t*>(dst)[lane] = E::pack(acc[0] * inv, acc[1] * inv);
        else
            dst[lane] = (uint16_t)E::pack(acc[0] * inv, 0.f);
        return;
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc_s[w][VPL * lane + i] = acc[i];
    __syncthreads();
    if (threadIdx.x < D / 2) {
        const int d = 2 * threadIdx.x;
        const float y0 = (acc_s[0][d] + acc_s[1][d]) + (acc_s[2][d] + acc_s[3][d]);
        const float y1 = (acc_s[0][d + 1] + acc_s[1][d + 1]) + (acc_s[2][d + 1] + acc_s[3][d + 1]);
        reinterpret_cast<uint32_t*>(dst)[threadIdx.x] = E::pack(y0 * inv, y1 * inv);
    }
}

struct SharedPlan {
    int workgroups, height, head_tiles;
    long long slots, rows;  // partial results of own rows, of prefix rows
};

SharedPlan shared_plan(int B, int qh, int kh) {
    SharedPlan p;
    const long long G = qh / kh;
    p.head_tiles = (int)((G + 15) / 16);
    p.workgroups = kWorkgroups / kh > 2 ? kWorkgroups / kh : 2;
    // Tiles of 64 rows, two waves to a row, while there are few.  64 / 128: 64 sequences of 32 / 8 heads over 4096 shared rows and
    // 30 to 1500 of their own 37.8 / 42.8 us, over 16384 73 / 70, over 16384 and one 57.0 / 56.7.
    p.height = B * G * kh <= 4096 ? 64 : 128;
    p.slots = 4ll * p.workgroups + B;
    p.rows = B * G + (long long)p.workgroups * p.height;
    return p;
}

template <typename E, int D, int KS, typename T, typename S>
int launch_shared(const SharedArgs& s, const typename S::Cache& c, const PagedBatch& bt, const SharedPlan& p, hipStream_t st) {
    const long long page = ((long long)c.kh << c.shift) * D * (std::is_same<typename S::Cache, PagedCache>::value ? 2 : 1);
    const long long named = (long long)bt.B * bt.W;
    const dim3 grid((unsigned)(p.workgroups * c.kh));
    if ((named < c.pages ? named : c.pages) * page * 2 > kCached)
        hipLaunchKernelGGL((paged_shared_split<E, D, KS, S, T, true>), grid, dim3(256), 0, st, s, c, bt);
    else
        hipLaunchKernelGGL((paged_shared_split<E, D, KS, S, T, false>), grid, dim3(256), 0, st, s, c, bt);
    // A sequence of few has many parts.  A wave a head / four: 2 sequences of 4200 own rows 24.8 / 19.0 us, 4 of 700 11.5 / 11.2, 16
    // over 4096 shared rows 21.2 / 20.8, 64 of 30 to 1500 own rows 27.5 / 29.2.
    if (bt.B <= 16)
        hipLaunchKernelGGL((paged_shared_join<E, D, 128 / KS, 4>), dim3((unsigned)s.a.qh, (unsigned)bt.B), dim3(256), 0, st, s);
    else
        hipLaunchKernelGGL((paged_shared_join<E, D, 128 / KS, 1>), dim3((unsigned)(s.a.qh + 3) / 4, (unsigned)bt.B), dim3(256), 0, st, s);
    return moss_launch_status();
}

template <typename E, int D, template <typename, int> class T, template <typename, int> class S, typename Cache>
int launch_shared(const SharedArgs& s, const Cache& c, const PagedBatch& bt, const SharedPlan& p, hipStream_t st) {
    return p.height == 64 ? launch_shared<E, D, 2, T<E, D>, S<E, D>>(s, c, bt, p, st) : launch_shared<E, D, 1, T<E, D>, S<E, D>>(s, c, bt, p, st);
}

long long workspace_bytes_of(const SharedPlan& p, int B, int qh, int kh, int d) {
    return (p.slots * qh + p.rows * kh) * (d + 2) * 4 + B * (long long)sizeof(Found);
}

template <template <typename, int> class T, template <typename, int> class S, typename Cache>
int shared_decode(const void* q, long long q_stride, const Cache& c, const PagedBatch& bt, const void* groups, const void* shared,
                  int qh, int d, float scale, void* out, void* workspace, long long workspace_bytes, int dtype, void* stream) {
    MOSS_CHECK_ARG(q && out && workspace && groups && shared && paged_pointers_ok(c, bt) && paged_shape_ok(c, bt, qh, d));
    MOSS_CHECK_ARG((dtype == 0 || dtype == 1) && q_stride % 8 == 0 && q_stride >= (long long)qh * d && paged_scale_ok(scale));
    MOSS_CHECK_ARG(MOSS_ALIGNED(q, 16) && MOSS_ALIGNED(out, 16) && MOSS_ALIGNED(workspace, 16) && MOSS_ALIGNED(groups, 4) &&
                   MOSS_ALIGNED(shared, 4));
    const SharedPlan p = shared_plan(bt.B, qh, c.kh);
    MOSS_CHECK_ARG(workspace_bytes >= workspace_bytes_of(p, bt.B, qh, c.kh, d));
    const long long own = p.slots * qh, rows = p.rows * c.kh;
    float* part = (float*)workspace;
    float* prefix_part = part + own * d;
    float2* stat = reinterpret_cast<float2*>(prefix_part + rows * d);
    // the scale is positive in either half, its sign goes to q; never 0, so a masked score stays -inf
    const DecodeArgs a{(const uint16_t*)q, q_stride, (uint16_t*)out, part, stat, qh, qh / c.kh, 0, 0, p.slots,
                       fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f), scale < 0.f ? 0x80008000u : 0u};
    const SharedArgs s{a, (const int*)groups, (const int*)shared, prefix_part, stat + own, p.rows, reinterpret_cast<Found*>(stat + own + rows), (kWorth / 16 + c.kh - 1) / c.kh, p.workgroups, p.head_tiles};
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
    return workspace_bytes_of(shared_plan(B, qh, kh), B, qh, kh, d);
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
