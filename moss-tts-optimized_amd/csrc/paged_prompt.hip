// Causal attention of packed prompts over a paged cache, on the matrix cores.
//
// The T packed tokens belong to B sequences (starts[b] .. starts[b + 1] - 1); token i of a sequence's n stands at
// position length - n + i and attends the rows 0 .. position of its sequence's pages, the cached ones before it and
// the new ones up to itself (all written).  o_h = sum_t softmax_t(scale q_h . k_t) v_t with query head h reading KV head
// h / (QH / KH); a token without a visible row gives zeros; tokens behind the last sequence are left alone.
//
// Tiling: the rows of a tile are (token, query head of the KV head's group) pairs, token first, so any group size fills
// them.  A workgroup takes 32 RW rows of one sequence and KV head; a wave takes 32 rows and, of every block of keys, the
// 32-key tiles ks, ks + KS, .. (SUB of them).  Which sequence and rows a workgroup has follows from starts on the device;
// the last rows, which see the most keys, go first.
//   S^T = K Q^T: 32 keys x 32 rows per matrix instruction, so a lane holds one row and 16 of its keys, and the row's
//   maximum needs one exchange with the lane 32 away; the running maximum and sum are fp32, base 2.
//   O^T += V^T P^T: P, rounded to 16 bits, is the B operand as S^T left it; V^T is read from LDS in the same K order.
// P's rounding is the one step with fewer bits before the output: the largest P of a tile is exactly 1 or its
// share of the running maximum, and the sum adds up the unrounded values.
// K / V blocks go from the pages through registers into two LDS stages (V transposed); block b + 2 is on its way while
// block b is consumed and b + 1 waits: one barrier per block.  The KS waves of the same rows are joined in LDS at the end.
#include "paged.h"

namespace moss {
namespace {

struct PromptArgs {
    const uint16_t* q;
    long long q_stride;
    uint16_t* out;
    int T, qh, group;
    float scale;    // |scale| log2(e), not 0: a masked score stays -inf
    uint32_t flip;  // its sign, for the two values of a word of q
};

template <int D, int RW, int KS, int SUB>
struct PromptTile {
    static constexpr int kRows = 32 * RW, kThreads = 64 * RW * KS;
    static constexpr int kBK = 32 * SUB * KS;                // keys per block
    static constexpr int kDC = D / 8;                        // 16-byte pieces of a row
    static constexpr int kKPT = kBK * kDC / kThreads;        // keys per thread in the copy
    static constexpr int kKPad = D + 8, kVPad = kBK + 4;     // LDS rows (16-bit values), padded
    static constexpr int kKBytes = kBK * kKPad * 2;
    static constexpr int kFlags = kKBytes + D * kVPad * 2;   // one byte per 16 keys: they have a page
    static constexpr int kStage = kFlags + 16;
    static constexpr int kXo = RW * (D / 32) * (KS - 1) * 4 * 64 * 16;  // O^T tiles handed over
    static constexpr int kMl = RW * KS * 2 * 64 * 4;
    static constexpr int kJoin = KS > 1 ? kXo + kMl : 0;
    static constexpr int kLds = 2 * kStage > kJoin ? 2 * kStage : kJoin;
    static_assert(kKPT == 1 || kKPT == 2 || kKPT == 4, "keys per thread in the copy");
    static_assert(kBK / 16 <= 16 && kKBytes % 16 == 0 && kStage % 16 == 0 && kXo % 16 == 0, "LDS layout");
    static_assert(kLds <= 160 * 1024, "LDS");
};

__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// V^T column of key `key` in row d: 8-key groups are swapped by XOR with 8 (d / 32), so the 16 rows that one store writes
// land in different banks; 4-key groups stay whole, and the rows of one read share d / 32.
__device__ __forceinline__ int vt_column(int d, int key) { return key ^ (8 * ((d >> 5) & 3)); }

template <typename E, int D, int RW, int KS, int SUB>
__global__ __launch_bounds__(64 * RW * KS, (RW * KS > 4 ? 1 : 2)) void paged_prompt_kernel(PromptArgs a, PagedCache c,
                                                                                           PagedBatch bt) {
    using T = PromptTile<D, RW, KS, SUB>;
    constexpr int KPT = T::kKPT, BK = T::kBK, KPAD = T::kKPad, VPAD = T::kVPad, DT = D / 32, DK = D / 16;
    __shared__ __attribute__((aligned(16))) unsigned char smem[T::kLds];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, rl = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rw = wave % RW, kq = wave / RW;
    const int kvh = blockIdx.x % c.kh, G = a.group;  // neighbours in the grid, which lie on different XCDs, differ in it
    const Place pl = find_item(bt.B, (int)((gridDim.x - 1 - blockIdx.x) / c.kh), lane, [&](int b) {
        return (int)(((long long)paged_tokens(bt, b, a.T).y * G + T::kRows - 1) / T::kRows);
    });
    if (pl.b < 0) return;
    const int2 tk = paged_tokens(bt, pl.b, a.T);
    const int len = paged_length(bt, pl.b, c.shift);
    const int pos0 = len - tk.y;  // position of the sequence's first new token (negative: it has none)
    const int row0 = pl.index * T::kRows, nrows = tk.y * G;
    const int row = min(row0 + 32 * rw + rl, nrows - 1);  // this lane's row (clamped: stores are guarded)
    const int token = row / G, head = kvh * G + row % G;
    const int qpos = pos0 + token;  // sees keys 0 .. qpos
    const int last = pos0 + min(row0 + T::kRows - 1, nrows - 1) / G;         // the workgroup's last key
    const int wave_last = pos0 + min(row0 + 32 * rw + 31, nrows - 1) / G;    // this wave's
    const int wave_first = pos0 + min(row0 + 32 * rw, nrows - 1) / G;        // keys up to it are seen by all its rows
    const int nblk = last / BK + (last >= 0 ? 1 : 0);

    auto stage_k = [&](int s) { return reinterpret_cast<uint16_t(*)[KPAD]>(smem + s * T::kStage); };
    auto stage_v = [&](int s) { return reinterpret_cast<uint16_t(*)[VPAD]>(smem + s * T::kStage + T::kKBytes); };
    auto stage_f = [&](int s) { return smem + s * T::kStage + T::kFlags; };

    u32x4_t qf[DK];  // lane: row rl, dims 16 kk + 8 half .. + 7
    {
        const uint16_t* qr = a.q + (size_t)(tk.x + token) * a.q_stride + (size_t)head * D + 8 * half;
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) qf[kk] = *reinterpret_cast<const u32x4_t*>(qr + 16 * kk) ^ a.flip;
    }
    f32x16_v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;

    // the copy: thread (kg, dc) holds keys KPT kg .. of a block (all in one 16-row group) at dims 8 dc .. + 7
    const int dc = tid % T::kDC, kg = tid / T::kDC;
    const int* trow = bt.table + (size_t)pl.b * bt.table_stride;
    auto page_of = [&](int b) {
        const int key = BK * b + KPT * kg;
        return key <= last ? page_or_none(trow[key >> c.shift], c.pages) : -1;
    };
    u32x4_t kr[KPT], vr[KPT];
    bool have = false;
    auto load = [&](int b, int page) {
        const int key = BK * b + KPT * kg;
        have = page >= 0;
        const uint16_t* kp = c.k + row_offset(page, c.k_stride, kvh, key, c.shift, D) + 8 * dc;
        const uint16_t* vp = c.v + row_offset(page, c.v_stride, kvh, key, c.shift, D) + 8 * dc;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            kr[i] = *reinterpret_cast<const u32x4_t*>(kp + (size_t)i * D);
            vr[i] = *reinterpret_cast<const u32x4_t*>(vp + (size_t)i * D);
        }
    };
    auto store = [&](int b) {
        uint16_t(*ks)[KPAD] = stage_k(b & 1);
        uint16_t(*vt)[VPAD] = stage_v(b & 1);
        const int key = BK * b + KPT * kg;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            *reinterpret_cast<u32x4_t*>(&ks[KPT * kg + i][8 * dc]) = kr[i];
            // rows that nobody sees may hold anything, and 0 times a NaN is one
            if (!have || key + i > last) vr[i] = u32x4_t{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            uint16_t* even = &vt[8 * dc + 2 * p][vt_column(8 * dc, KPT * kg)];
            uint16_t* odd = &vt[8 * dc + 2 * p + 1][vt_column(8 * dc, KPT * kg)];
            if constexpr (KPT == 4) {
                *reinterpret_cast<uint2*>(even) = make_uint2(low_halves(vr[0][p], vr[1][p]), low_halves(vr[2][p], vr[3][p]));
                *reinterpret_cast<uint2*>(odd) = make_uint2(high_halves(vr[0][p], vr[1][p]), high_halves(vr[2][p], vr[3][p]));
            } else if constexpr (KPT == 2) {
                *reinterpret_cast<uint32_t*>(even) = low_halves(vr[0][p], vr[1][p]);
                *reinterpret_cast<uint32_t*>(odd) = high_halves(vr[0][p], vr[1][p]);
            } else {
                *even = (uint16_t)vr[0][p];
                *odd = (uint16_t)(vr[0][p] >> 16);
            }
        }
        if (dc == 0 && (KPT * kg) % 16 == 0) stage_f(b & 1)[KPT * kg / 16] = have ? 1 : 0;
    };

    int page = -1;
    if (nblk > 0) {
        load(0, page_of(0));
        page = page_of(1);
        store(0);
        if (nblk > 1) {
            load(1, page);
            page = page_of(2);
        }
    }
    for (int b = 0; b < nblk; ++b) {
        // block b is staged by every wave, and every wave is done with block b - 1's stage
        __syncthreads();
        const uint16_t(*ks)[KPAD] = stage_k(b & 1);
        const uint16_t(*vt)[VPAD] = stage_v(b & 1);
        const unsigned char* flags = stage_f(b & 1);
        const int part = 32 * kq;
        if (BK * b + part <= wave_last) {  // else none of its rows sees any of its keys
            f32x16_v s[SUB];
#pragma unroll
            for (int i = 0; i < SUB; ++i) s[i] = f32x16_v{};
#pragma unroll
            for (int kk = 0; kk < DK; ++kk)
#pragma unroll
                for (int i = 0; i < SUB; ++i) {
                    const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(&ks[part + 32 * KS * i + rl][16 * kk + 8 * half]);
                    s[i] = E::mfma32(kf, qf[kk], s[i]);
                }
            // element e of tile i: key BK b + part + 32 KS i + 8 (e / 4) + 4 half + e % 4, row rl
            bool holes = false;
#pragma unroll
            for (int i = 0; i < SUB; ++i) {
                const int f = (part + 32 * KS * i) / 16;
                holes |= !(flags[f] & flags[f + 1]);
            }
            if (__any(holes) || BK * b + BK - 1 > wave_first) {
#pragma unroll
                for (int i = 0; i < SUB; ++i) {
                    const int tile = part + 32 * KS * i;
                    const bool f0 = flags[tile / 16], f1 = flags[tile / 16 + 1];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int key = BK * b + tile + 8 * (e >> 2) + 4 * half + (e & 3);
                        s[i][e] = key <= qpos && (e < 8 ? f0 : f1) ? s[i][e] : -INFINITY;
                    }
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < SUB; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[i][e]);
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
            for (int i = 0; i < SUB; ++i) {
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
                for (int u = 0; u < 2; ++u) {
                    const int key = part + 32 * KS * i + 16 * u + 4 * half;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const uint16_t* vrow = vt[32 * dt + rl];
                        const uint2 a0 = *reinterpret_cast<const uint2*>(vrow + vt_column(32 * dt, key));
                        const uint2 a1 = *reinterpret_cast<const uint2*>(vrow + vt_column(32 * dt, key + 8));
                        o[dt] = E::mfma32(u32x4_t{a0.x, a0.y, a1.x, a1.y}, pf[u], o[dt]);
                    }
                }
            }
        }
        if (b + 1 < nblk) {  // block b + 1's stage was last read for block b - 1
            store(b + 1);
            if (b + 2 < nblk) {
                load(b + 2, page);
                page = page_of(b + 3);
            }
        }
    }
    l = sum_xor32(l);
    float inv;
    if constexpr (KS == 1) {
        inv = l == 0.f ? 0.f : 1.0f / l;
    } else {
        // each of a row's KS waves finishes the d tiles dt with dt % KS == kq from all of them
        __syncthreads();
        float4* xo = reinterpret_cast<float4*>(smem);  // [RW][dt][KS - 1 slots][e / 4][lane]
        float* ml = reinterpret_cast<float*>(smem + T::kXo);
        ml[((rw * KS + kq) * 2) * 64 + lane] = m;
        ml[((rw * KS + kq) * 2 + 1) * 64 + lane] = l;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int owner = dt % KS;
            if (owner == kq) continue;
            const int slot = kq < owner ? kq : kq - 1;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                xo[(((rw * DT + dt) * (KS - 1) + slot) * 4 + j) * 64 + lane] =
                    make_float4(o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]);
        }
        __syncthreads();
        float f[KS], mx = -INFINITY, den = 0.f;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            f[j] = ml[((rw * KS + j) * 2) * 64 + lane];
            mx = fmaxf(mx, f[j]);
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            f[j] = f[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(f[j] - mx);
            den = fmaf(ml[((rw * KS + j) * 2 + 1) * 64 + lane], f[j], den);
        }
        inv = den == 0.f ? 0.f : 1.0f / den;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int owner = dt % KS;
            if (owner != kq) continue;
#pragma unroll
            for (int j4 = 0; j4 < 4; ++j4) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    float4 w;
                    if (j == kq) {
                        w = make_float4(o[dt][4 * j4], o[dt][4 * j4 + 1], o[dt][4 * j4 + 2], o[dt][4 * j4 + 3]);
                    } else {
                        const int slot = j < owner ? j : j - 1;
                        w = xo[(((rw * DT + dt) * (KS - 1) + slot) * 4 + j4) * 64 + lane];
                    }
                    acc[0] = fmaf(w.x, f[j], acc[0]);
                    acc[1] = fmaf(w.y, f[j], acc[1]);
                    acc[2] = fmaf(w.z, f[j], acc[2]);
                    acc[3] = fmaf(w.w, f[j], acc[3]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) o[dt][4 * j4 + i] = acc[i];
            }
        }
    }
    if (row0 + 32 * rw + rl >= nrows) return;
    uint16_t* dst = a.out + ((size_t)(tk.x + token) * a.qh + head) * D;
    // O^T element e of d tile dt: d = 32 dt + 8 (e / 4) + 4 half + e % 4
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        if (dt % KS != kq) continue;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<uint2*>(dst + 32 * dt + 8 * q4 + 4 * half) =
                make_uint2(E::pack(o[dt][4 * q4] * inv, o[dt][4 * q4 + 1] * inv),
                           E::pack(o[dt][4 * q4 + 2] * inv, o[dt][4 * q4 + 3] * inv));
    }
}

template <typename E, int D, int RW, int KS, int SUB>
int launch_prompt_tile(const PromptArgs& a, const PagedCache& c, const PagedBatch& bt, hipStream_t st) {
    using T = PromptTile<D, RW, KS, SUB>;
    const long long groups = (((long long)a.T * a.group + T::kRows - 1) / T::kRows + bt.B) * c.kh;
    MOSS_CHECK_ARG(groups * T::kThreads < (1ll << 32));
    hipLaunchKernelGGL((paged_prompt_kernel<E, D, RW, KS, SUB>), dim3((unsigned)groups), dim3(T::kThreads), 0, st, a, c,
                       bt);
    return moss_launch_status();
}

template <typename E, int D>
int launch_prompt(const PromptArgs& a, const PagedCache& c, const PagedBatch& bt, hipStream_t st) {
    const long long rows = (long long)a.T * a.group * c.kh;  // rows over all KV heads
    if (rows <= 32 * 512) return launch_prompt_tile<E, D, 2, 2, 1>(a, c, bt, st);
    return launch_prompt_tile<E, D, 4, 1, 2>(a, c, bt, st);
}

}  // namespace
}  // namespace moss

using namespace moss;

MOSS_API int moss_paged_prompt_attention(const void* q, long long q_stride, const void* k, const void* v,
                                         long long k_stride, long long v_stride, int pages, int page_rows,
                                         const void* table, long long table_stride, const void* lengths,
                                         const void* starts, int B, int W, int T, int qh, int kh, int d, float scale,
                                         void* out, int dtype, void* stream) {
    const PagedCache c = paged_cache(k, v, k_stride, v_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, (const int*)starts, B, W, table_stride};
    MOSS_CHECK_ARG(q && out && starts && paged_pointers_ok(c, bt) && paged_shape_ok(c, bt, qh, d));
    MOSS_CHECK_ARG((dtype == 0 || dtype == 1) && T > 0 && T <= (1 << 20) && q_stride % 8 == 0 &&
                   q_stride >= (long long)qh * d && scale == scale);
    MOSS_CHECK_ARG(MOSS_ALIGNED(q, 16) && MOSS_ALIGNED(out, 16));
    const PromptArgs a{(const uint16_t*)q, q_stride, (uint16_t*)out, T, qh, qh / kh, fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f),
                       scale < 0.f ? 0x80008000u : 0u};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0) return d == 128 ? launch_prompt<Bf16, 128>(a, c, bt, st) : launch_prompt<Bf16, 64>(a, c, bt, st);
    return d == 128 ? launch_prompt<F16, 128>(a, c, bt, st) : launch_prompt<F16, 64>(a, c, bt, st);
}
