// Kernels of branching histories (include/kvl/mla_hip.h): the attention of a tree of drafted tokens
// over a latent history, copies of a state's rows, and the compaction of an accepted path's rows.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mla_device.h"
#include "mla_internal.h"

namespace kvl {

// ================================================================ tree attention =======

// Node i of a tree over a history of n rows (row n + i is its own) attends rows 0 .. n - 1, the rows
// of its ancestors and its own, in one softmax per head:
//   s_j = (q_lat . lat_j + q_rope . key_j) / sqrt(QD),  mix = sum_j softmax(s)_j lat_j.
// Rows of other branches are never read for it, so nothing they hold (NaN, infinities) reaches it.

template <int FMT>
__device__ __forceinline__ float tree_lat(const TreeSeq &s, size_t row, int R, int k) {
    if (FMT == kFmtQ8) return (float)((const int8_t *)s.a)[row * R + k] * ((const float *)s.b)[row];
    if (FMT == kFmtF32) return ((const float *)s.a)[row * R + k];
    return bf16_to_f32(((const uint16_t *)s.a)[row * R + k]);
}
template <int FMT>
__device__ __forceinline__ float tree_key(const TreeSeq &s, size_t row, int DR, int k) {
    if (FMT == kFmtQ8) return bf16_to_f32(((const uint16_t *)s.c)[row * DR + k]);
    if (FMT == kFmtF32) return ((const float *)s.b)[row * DR + k];
    return bf16_to_f32(((const uint16_t *)s.b)[row * DR + k]);
}

struct TreeArgs {
    TreeTable t;
    Dims d;
    const float *qf;
    float *part;
    float smscale;
};

constexpr int kTgRows = 256;  // rows taken at a time: a thread per row
constexpr int kTgCols = 4;    // latent columns per thread: R <= 1024

// Any dims: one workgroup per (node, head) goes over the node's rows kTgRows at a time with the
// running maximum and sum of the softmax; a thread per row forms the scores, a thread per latent
// column the mix.
template <int FMT>
__global__ __launch_bounds__(256) void k_tree_generic(TreeArgs a) {
    __shared__ float q[1024 + 256];
    __shared__ float p[kTgRows];
    __shared__ float redm[4], reds[4];
    __shared__ int path[kTreeNodes];
    __shared__ int npath;
    const int tid = threadIdx.x, NH = a.d.NH, R = a.d.R, DR = a.d.DR;
    const int k = blockIdx.x / NH, h = blockIdx.x % NH;
    const TreeSeq s = a.t.s[a.t.seq[k]];
    for (int i = tid; i < R + DR; i += 256) q[i] = a.qf[((size_t)k * NH + h) * (R + DR) + i];
    if (tid == 0) {  // the node and its ancestors, in the order of their rows
        int n = 0;
        for (int i = k - s.node0; i >= 0; i = a.t.parent[s.node0 + i]) ++n;
        npath = n;
        for (int i = k - s.node0; i >= 0; i = a.t.parent[s.node0 + i]) path[--n] = i;
    }
    __syncthreads();
    const int rows = s.ctx + npath;
    float m = -INFINITY, l = 0.f, acc[kTgCols] = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < rows; j0 += kTgRows) {
        const int j = j0 + tid;
        float sc = -INFINITY;
        if (j < rows) {
            const size_t row = j < s.ctx ? (size_t)j : (size_t)s.ctx + path[j - s.ctx];
            float v = 0.f;
            for (int i = 0; i < R; ++i) v = fmaf(q[i], tree_lat<FMT>(s, row, R, i), v);
            for (int i = 0; i < DR; ++i) v = fmaf(q[R + i], tree_key<FMT>(s, row, DR, i), v);
            sc = v * a.smscale;
        }
        const float cm = block256_max(sc, redm);  // -inf only if every score is (or is NaN)
        const float mn = fmaxf(m, cm);
        const float ref = mn == -INFINITY ? 0.f : mn;  // exp(-inf - -inf) is NaN
        const float e = j < rows ? __expf(sc - ref) : 0.f;
        p[tid] = e;
        const float ws = wave_sum(e);
        if ((tid & 63) == 0) reds[tid >> 6] = ws;
        __syncthreads();
        const float alpha = m == -INFINITY ? 0.f : __expf(m - ref);
        l = l * alpha + ((reds[0] + reds[1]) + (reds[2] + reds[3]));
        m = mn;
        const int n = min(kTgRows, rows - j0);
#pragma unroll
        for (int c = 0; c < kTgCols; ++c) {
            const int col = tid + 256 * c;
            if (col >= R) break;
            float v = acc[c] * alpha;
            for (int i = 0; i < n; ++i) {
                const size_t row = j0 + i < s.ctx ? (size_t)(j0 + i) : (size_t)s.ctx + path[j0 + i - s.ctx];
                v = fmaf(p[i], tree_lat<FMT>(s, row, R, col), v);
            }
            acc[c] = v;
        }
        __syncthreads();  // p and the reductions are rewritten
    }
    float *P = a.part + (size_t)k * NH * (R + 2);
#pragma unroll
    for (int c = 0; c < kTgCols; ++c)
        if (tid + 256 * c < R) P[(size_t)h * R + tid + 256 * c] = acc[c];
    if (tid == 0) {
        P[(size_t)NH * R + h] = m;
        P[(size_t)NH * R + NH + h] = l;
    }
}

// ---- the tree's own rows (Kimi shapes: NH = 16, R = 512, DR = 64) ----------------------------------

// One workgroup of eight waves per node, wave w its heads 2w, 2w + 1, lane l columns l + 64 q and key
// column l: the scores of the node's path (at most 64 rows: row j's in lane j), their maximum and
// weights, then the mix. fp32 throughout. The partial after the node's history partials.
template <int FMT>
__global__ __launch_bounds__(512) void k_tree_path(TreeArgs a) {
    constexpr int R = 512, DR = 64, NH = 16;
    __shared__ int path[kTreeNodes];
    __shared__ int npath;
    const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), k = blockIdx.x;
    const TreeSeq s = a.t.s[a.t.seq[k]];
    if (tid == 0) {
        int n = 0;
        for (int i = k - s.node0; i >= 0; i = a.t.parent[s.node0 + i]) ++n;
        npath = n;
        for (int i = k - s.node0; i >= 0; i = a.t.parent[s.node0 + i]) path[--n] = i;
    }
    float q[2][9];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 9; ++c) q[h][c] = a.qf[((size_t)k * NH + 2 * w + h) * (R + DR) + 64 * c + l] * a.smscale;
    __syncthreads();
    const int n = npath;
    float sc[2] = {-INFINITY, -INFINITY};
    for (int j = 0; j < n; ++j) {
        const size_t row = (size_t)s.ctx + path[j];
        float v0 = 0.f, v1 = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float x = tree_lat<FMT>(s, row, R, 64 * c + l);
            v0 = fmaf(q[0][c], x, v0);
            v1 = fmaf(q[1][c], x, v1);
        }
        const float x = tree_key<FMT>(s, row, DR, l);
        v0 = wave_sum(fmaf(q[0][8], x, v0));
        v1 = wave_sum(fmaf(q[1][8], x, v1));
        if (l == j) {
            sc[0] = v0;
            sc[1] = v1;
        }
    }
    float m[2], p[2], sum[2], acc[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        m[h] = wave_max(sc[h]);
        p[h] = l < n ? __expf(sc[h] - m[h]) : 0.f;
        sum[h] = wave_sum(p[h]);
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[h][c] = 0.f;
    }
    for (int j = 0; j < n; ++j) {
        const size_t row = (size_t)s.ctx + path[j];
        const float p0 = lane_f32(p[0], j), p1 = lane_f32(p[1], j);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float x = tree_lat<FMT>(s, row, R, 64 * c + l);
            acc[0][c] = fmaf(p0, x, acc[0][c]);
            acc[1][c] = fmaf(p1, x, acc[1][c]);
        }
    }
    float *P = a.part + (size_t)(s.part0 + (k - s.node0) * (s.ns + 1) + s.ns) * NH * (R + 2);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < 8; ++c) P[(2 * w + h) * R + 64 * c + l] = acc[h][c];
        if (l == 0) {
            P[NH * R + 2 * w + h] = m[h];
            P[NH * R + NH + 2 * w + h] = sum[h];
        }
    }
}

// ---- the history (Kimi shapes) ------------------------------------------------------------------

// A workgroup takes NM nodes of one tree (16 NM queries) over one split of the history, in chunks of 32
// rows that all its waves share in LDS: 2 NM waves,
//   scores: wave (m, kh) = node m's 16 heads x 32 rows over half kh of the 576 columns, the queries held
//     in registers; the two halves are added through LDS;
//   softmax: 8 threads per query, 4 rows each, running maximum (moved only when a chunk exceeds it by
//     more than ln 4) and sum in registers; weights to LDS as the next product's operand;
//   mix: every wave 512 / (2 NM) latent columns of all 16 NM queries, the rows read transposed.
// Operands are 16 bits wide, sums 32: the 32-bit query and weight enter as hi + lo (two products), the
// BF16 rows as they are, the FP32 rows as hi + lo too (without lo . lo: three products), all in bf16 (what
// is left out is below 2^-17 of an operand). Q8 codes are exact in fp16, so there the query (times a
// power of two that puts its largest element near 2^10) and the weights are split in fp16, which keeps 22
// bits. A Q8 row's scale multiplies its latent score and its weight; to keep the weights within fp16
// whatever the scales, the running maximum is that of score + ln(scale), so that weight times scale stays
// <= 4.
constexpr int kThCh = 32;       // rows of a chunk
constexpr int kThSp = 36;       // floats per query in a score half
constexpr int kThPw = 80;       // bytes per query in a weight plane (32 bf16, padded)
template <int FMT, int NM>
struct ThShape {
    static constexpr int NW = 2 * NM, NT = 64 * NW, NQ = 16 * NM;
    static constexpr int NP = FMT == kFmtF32 ? 2 : 1;  // planes of a row
    static constexpr int LatB = kThCh * 1024, KeyB = kThCh * 128, PlaneB = LatB + KeyB;
    static constexpr int ScB = FMT == kFmtQ8 ? 2 * kThCh * 4 : 0;  // scales, their logarithms
    static constexpr int Slot = NP * PlaneB + ScB;
    static constexpr int Ring = FMT == kFmtF32 || NM < 4 ? 1 : 2;
    static constexpr int SpOff = Ring * Slot;
    static constexpr int PwOff = SpOff + 2 * NQ * kThSp * 4;
    static constexpr int AlOff = PwOff + 2 * NQ * kThPw;
    static constexpr int FlOff = AlOff + NQ * 4;
    static constexpr int Smem = FlOff + 2 * 8 * 4;
    static_assert(Smem <= 160 * 1024, "LDS of one CU");
};

// Workgroup -> (sequence, split, tile). Workgroup i runs on XCD i % 8; the units (a sequence's split) go
// to the XCDs in turn, and the tiles of a unit follow one another on its XCD, so that its L2 serves the
// rows they share. Lane b of every wave counts what sequence b has on this XCD.
__device__ __forceinline__ bool tree_unit(const TreeTable &t, int &b, int &split, int &tile) {
    const int lane = threadIdx.x & 63, xcd = blockIdx.x & 7, j = blockIdx.x >> 3;
    const TreeSeq &q = t.s[lane];
    const int live = lane < t.n ? 1 : 0, u0 = live ? q.unit0 : 0, ns = live ? q.ns : 0, tiles = live ? q.tiles : 0;
    const int first = (xcd - u0) & 7;  // the first of its splits on this XCD
    const int mine = (ns > first ? (ns - first + 7) / 8 : 0) * tiles;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(sum, o);
        if (lane >= o) sum += v;
    }
    if (j >= __shfl(sum, 63)) return false;
    b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(sum <= j));
    const int r = j - __shfl(sum - mine, b), tl = __shfl(tiles, b);
    split = __shfl(first, b) + 8 * (r / tl);
    tile = r % tl;
    b = __builtin_amdgcn_readfirstlane(b);
    split = __builtin_amdgcn_readfirstlane(split);
    tile = __builtin_amdgcn_readfirstlane(tile);
    return true;
}

template <int FMT>
__device__ __forceinline__ v4f th_mfma(const v4i &a, const v4i &b, const v4f &c) {
    if (FMT == kFmtQ8) return mfma_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c);
    return mfma_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c);
}

// Eight fp32 values as hi and lo operands: bf16, or fp16 for the latents of Q8.
template <bool F16>
__device__ __forceinline__ void th_split(const v4f &x0, const v4f &x1, v4i &hi, v4i &lo) {
    if constexpr (F16) {
        const float x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
        v8h h, r;
        split8_f16(x, h, r);
        hi = __builtin_bit_cast(v4i, h);
        lo = __builtin_bit_cast(v4i, r);
    } else {
        v8bf h, r;
        split8_cvt(x0, x1, h, r);
        hi = __builtin_bit_cast(v4i, h);
        lo = __builtin_bit_cast(v4i, r);
    }
}

// Sixteen int8 codes -> sixteen fp16 values, exact: the code + 128 as the low mantissa bits of 1024,
// minus 1152.
__device__ __forceinline__ void codes_f16(const v4i &c, v4i &o0, v4i &o1) {
    const v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = (uint32_t)c[i] ^ 0x80808080u;
        const uint32_t a = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
        const uint32_t b = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
        o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, a) - off);
        o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, b) - off);
    }
    o0 = v4i{(int)o[0], (int)o[1], (int)o[2], (int)o[3]};
    o1 = v4i{(int)o[4], (int)o[5], (int)o[6], (int)o[7]};
}

template <int FMT, int NM>
__global__ __launch_bounds__(128 * NM) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_tree_hist(TreeArgs a) {
    using Sh = ThShape<FMT, NM>;
    constexpr int NT = Sh::NT, NW = Sh::NW, NQ = Sh::NQ, NP = Sh::NP, Ring = Sh::Ring;
    constexpr int NC = 512 / NW / 16;  // 16-column blocks of a wave in the mix
    constexpr bool kQ8 = FMT == kFmtQ8;
    __shared__ __attribute__((aligned(16))) uint8_t smem[Sh::Smem];
    const int tid = threadIdx.x, l = tid & 63, n = l & 15, g = l >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int b, split, tile;
    if (!tree_unit(a.t, b, split, tile)) return;
    const TreeSeq &s = a.t.s[b];
    const int r0 = split * s.rps, r1 = split == s.ns - 1 ? s.ctx : r0 + s.rps;
    const int nch = (r1 - r0 + kThCh - 1) / kThCh;
    const int first = tile * NM, live = min(NM, s.count - first);  // nodes of this tile
    float *sp = (float *)(smem + Sh::SpOff);

    // ---- staging: a chunk's rows from memory to registers, and from there to an LDS slot. Row j's
    // 16-byte word c lies at word c ^ b16_swz(j) of its latents, c ^ (j & 7) of its key. Rows past the
    // split's end repeat its last row (their scores are masked).
    constexpr int NL = (kQ8 ? 1024 : 2048) / NT;  // latent items of a thread (16 codes, or 8 values)
    constexpr int NK = (256 + NT - 1) / NT;       // key items (8 values)
    v4i la[NL], lb[FMT == kFmtF32 ? NL : 1], ka[NK], kb[FMT == kFmtF32 ? NK : 1];
    float rsc = 0.f;
    auto fetch = [&](int c) __attribute__((always_inline)) {
        const int base = r0 + c * kThCh;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int it = tid + NT * i;
            if constexpr (kQ8) {
                la[i] = *(const v4i *)((const int8_t *)s.a + (size_t)min(base + (it >> 5), r1 - 1) * 512 + 16 * (it & 31));
            } else if constexpr (FMT == kFmtF32) {
                const float *p = (const float *)s.a + (size_t)min(base + (it >> 6), r1 - 1) * 512 + 8 * (it & 63);
                la[i] = *(const v4i *)p;
                lb[i] = *(const v4i *)(p + 4);
            } else {
                la[i] = *(const v4i *)((const uint16_t *)s.a + (size_t)min(base + (it >> 6), r1 - 1) * 512 + 8 * (it & 63));
            }
        }
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int it = tid + NT * i;
            if (it < 256) {
                const size_t row = (size_t)min(base + (it >> 3), r1 - 1);
                if constexpr (FMT == kFmtF32) {
                    const float *p = (const float *)s.b + row * 64 + 8 * (it & 7);
                    ka[i] = *(const v4i *)p;
                    kb[i] = *(const v4i *)(p + 4);
                } else {
                    ka[i] = *(const v4i *)((const uint16_t *)(kQ8 ? s.c : s.b) + row * 64 + 8 * (it & 7));
                }
            }
        }
        if constexpr (kQ8) rsc = ((const float *)s.b)[min(base + (tid & 31), r1 - 1)];
    };
    auto stage = [&](int c) __attribute__((always_inline)) {
        uint8_t *buf = smem + (c % Ring) * Sh::Slot;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int it = tid + NT * i;
            if constexpr (kQ8) {
                const int row = it >> 5, word = 2 * (it & 31), z = b16_swz(row);
                v4i o0, o1;
                codes_f16(la[i], o0, o1);
                *(v4i *)(buf + row * 1024 + 16 * (word ^ z)) = o0;
                *(v4i *)(buf + row * 1024 + 16 * ((word + 1) ^ z)) = o1;
            } else {
                const int row = it >> 6, at = row * 1024 + 16 * ((it & 63) ^ b16_swz(row));
                if constexpr (FMT == kFmtF32) {
                    v4i hi, lo;
                    th_split<false>(__builtin_bit_cast(v4f, la[i]), __builtin_bit_cast(v4f, lb[i]), hi, lo);
                    *(v4i *)(buf + at) = hi;
                    *(v4i *)(buf + Sh::PlaneB + at) = lo;
                } else {
                    *(v4i *)(buf + at) = la[i];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int it = tid + NT * i;
            if (it < 256) {
                const int row = it >> 3, at = Sh::LatB + row * 128 + 16 * ((it & 7) ^ (row & 7));
                if constexpr (FMT == kFmtF32) {
                    v4i hi, lo;
                    th_split<false>(__builtin_bit_cast(v4f, ka[i]), __builtin_bit_cast(v4f, kb[i]), hi, lo);
                    *(v4i *)(buf + at) = hi;
                    *(v4i *)(buf + Sh::PlaneB + at) = lo;
                } else {
                    *(v4i *)(buf + at) = ka[i];
                }
            }
        }
        if constexpr (kQ8) {
            if (tid < kThCh) {
                float *sc = (float *)(buf + NP * Sh::PlaneB);
                sc[tid] = rsc;
                sc[kThCh + tid] = __logf(fmaxf(fabsf(rsc), 1e-35f));
            }
        }
    };

    fetch(0);
    // ---- queries: A operand of the scores, head n of node m, columns 32 kb + 8 g ..
    const int m = w % NM, kh = w / NM;
    v4i qh[9], ql[9];
    float qi = 1.0f;  // Q8: undoes the query's power of two, per head 4 g + i below
    float qd[4] = {1.f, 1.f, 1.f, 1.f};
    {
        const float *qrow = a.qf + ((size_t)(s.node0 + first + min(m, live - 1)) * 16 + n) * 576 + 8 * g;
        v4f qv[18];
#pragma unroll
        for (int j = 0; j < 9; ++j) {
            qv[2 * j] = *(const v4f *)(qrow + 32 * (9 * kh + j));
            qv[2 * j + 1] = *(const v4f *)(qrow + 32 * (9 * kh + j) + 4);
        }
        float qs = a.smscale;
        if constexpr (kQ8) {
            float mx = 0.f;
#pragma unroll
            for (int j = 0; j < 18; ++j)
                if (kh == 0 || j < 14)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(qv[j][e]));
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            mx *= a.smscale;
            // 2^(10 - e) with 2^(e - 1) <= mx < 2^e, kept within the normal exponents
            const int e = mx > 0.f && mx < INFINITY ? min(max(ilogbf(mx) + 1, -100), 100) : 10;
            qs = ldexpf(a.smscale, 10 - e);
            qi = ldexpf(1.0f, e - 10);
#pragma unroll
            for (int i = 0; i < 4; ++i) qd[i] = __shfl(qi, 4 * g + i);
        }
#pragma unroll
        for (int j = 0; j < 9; ++j) {
            if (kQ8 && (kh == 0 || j < 7)) th_split<true>(qv[2 * j] * qs, qv[2 * j + 1] * qs, qh[j], ql[j]);
            else th_split<false>(qv[2 * j] * a.smscale, qv[2 * j + 1] * a.smscale, qh[j], ql[j]);
        }
    }
    stage(0);
    if (nch > 1) fetch(1);

    // score operands: row n of a 16-row half (16 KB / 2 KB apart), words 4 kb + g
    int bofs[9];
#pragma unroll
    for (int j = 0; j < 9; ++j) {
        const int kb = 9 * kh + j;
        bofs[j] = kb < 16 ? n * 1024 + 16 * ((4 * kb + g) ^ b16_swz(n)) : Sh::LatB + n * 128 + 16 * ((4 * (kb - 16) + g) ^ (n & 7));
    }
    // transposed reads of column block NC w + t: rows 8 g + 4 h + (n >> 2), see lds_read_tr16
    int tro[2][NC];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = 8 * g + 4 * h + (n >> 2);
#pragma unroll
        for (int t = 0; t < NC; ++t)
            tro[h][t] = row * 1024 + 16 * ((2 * (NC * w + t) + ((n >> 1) & 1)) ^ b16_swz(row)) + 8 * (n & 1);
    }
    const int sq = tid >> 3, sr = 4 * (tid & 7);  // softmax: this thread's query and rows
    float m_run = -INFINITY, l_run = 0.f;
    v4f acc[NM][NC];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int t = 0; t < NC; ++t) acc[i][t] = v4f{0.f, 0.f, 0.f, 0.f};
    lds_barrier();

    for (int c = 0; c < nch; ++c) {
        const uint8_t *buf = smem + (c % Ring) * Sh::Slot;
        const float *scl = (const float *)(buf + NP * Sh::PlaneB);
        // ---- scores
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
            v4f dl = {0.f, 0.f, 0.f, 0.f}, dk = {0.f, 0.f, 0.f, 0.f};  // over latents, over the key
#pragma unroll
            for (int j = 0; j < 9; ++j) {
                const bool key = j >= 7 && kh == 1;
                const uint8_t *p = buf + bofs[j] + (j >= 7 && kh == 1 ? rb * 2048 : rb * 16384);
                const v4i bv = *(const v4i *)p;
                if (kQ8 && key) {
                    dk = th_mfma<kFmtBF16>(qh[j], bv, dk);
                    dk = th_mfma<kFmtBF16>(ql[j], bv, dk);
                } else {
                    dl = th_mfma<FMT>(qh[j], bv, dl);
                    dl = th_mfma<FMT>(ql[j], bv, dl);
                }
                if constexpr (NP == 2) dl = th_mfma<FMT>(qh[j], *(const v4i *)(p + Sh::PlaneB), dl);
            }
            if constexpr (kQ8) {
                const float x = scl[16 * rb + n];
#pragma unroll
                for (int i = 0; i < 4; ++i) dl[i] = fmaf(dl[i], qd[i] * x, dk[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sp[(size_t)(kh * NQ + 16 * m + 4 * g + i) * kThSp + 16 * rb + n] = dl[i];
        }
        lds_barrier();  // both halves of every score are in LDS
        // ---- softmax
        {
            const v4f s0 = *(const v4f *)(sp + sq * kThSp + sr), s1 = *(const v4f *)(sp + (NQ + sq) * kThSp + sr);
            const int nv = r1 - (r0 + c * kThCh) - sr;  // of this thread's rows, the ones in the split
            v4f x, t, rs;
            if constexpr (kQ8) {
                rs = *(const v4f *)(scl + sr);
                t = *(const v4f *)(scl + kThCh + sr);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = e < nv ? s0[e] + s1[e] : -INFINITY;
                t[e] = kQ8 ? x[e] + t[e] : x[e];
            }
            float cm = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
            cm = fmaxf(cm, dpp_f32<0xB1>(cm));
            cm = fmaxf(cm, dpp_f32<0x4E>(cm));
            cm = fmaxf(cm, dpp_f32<0x141>(cm));  // row_half_mirror: the other four of the eight
            const bool mv = cm > m_run + 1.3862944f;
            float alpha = 1.0f;
            if (mv) {
                alpha = __expf(m_run - cm);
                m_run = cm;
                l_run *= alpha;
            }
            if ((tid & 7) == 0) *(float *)(smem + Sh::AlOff + 4 * sq) = alpha;
            const bool any = __any(mv);
            if (l == 0) *(int *)(smem + Sh::FlOff + 32 * (c & 1) + 4 * w) = any ? 1 : 0;
            v4f p;
            float ps = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = __expf(x[e] - m_run);
                ps += p[e];
                if constexpr (kQ8) p[e] *= rs[e];
            }
            l_run += ps;  // this thread's rows; the eight threads' sums are added at the end
            v4i hi, lo;
            th_split<kQ8>(p, v4f{0.f, 0.f, 0.f, 0.f}, hi, lo);
            *(int2 *)(smem + Sh::PwOff + sq * kThPw + 2 * sr) = int2{hi[0], hi[1]};
            *(int2 *)(smem + Sh::PwOff + (NQ + sq) * kThPw + 2 * sr) = int2{lo[0], lo[1]};
        }
        if constexpr (Ring == 2) {
            if (c + 1 < nch) stage(c + 1);
            if (c + 2 < nch) fetch(c + 2);
        }
        lds_barrier();  // the weights (and the next chunk) are in LDS
        // ---- mix
        {
            int any = 0;
#pragma unroll
            for (int i = 0; i < NW / 4; ++i) {
                const v4i f = *(const v4i *)(smem + Sh::FlOff + 32 * (c & 1) + 16 * i);
                any |= f[0] | f[1] | f[2] | f[3];
            }
            if (__builtin_amdgcn_readfirstlane(any)) {
#pragma unroll
                for (int i = 0; i < NM; ++i) {
                    const v4f al = *(const v4f *)(smem + Sh::AlOff + 64 * i + 16 * g);
#pragma unroll
                    for (int t = 0; t < NC; ++t) acc[i][t] *= al;
                }
            }
            v4i ph[NM], pl[NM];
#pragma unroll
            for (int i = 0; i < NM; ++i) {
                ph[i] = *(const v4i *)(smem + Sh::PwOff + (16 * i + n) * kThPw + 16 * g);
                pl[i] = *(const v4i *)(smem + Sh::PwOff + (NQ + 16 * i + n) * kThPw + 16 * g);
            }
#pragma unroll
            for (int t = 0; t < NC; ++t) {
                v4i bt[NP];
#pragma unroll
                for (int z = 0; z < NP; ++z)
                    bt[z] = __builtin_bit_cast(v4i, __builtin_shufflevector(lds_read_tr16(buf + z * Sh::PlaneB + tro[0][t]),
                                                                            lds_read_tr16(buf + z * Sh::PlaneB + tro[1][t]), 0, 1,
                                                                            2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int i = 0; i < NM; ++i) {
                    acc[i][t] = th_mfma<FMT>(ph[i], bt[0], acc[i][t]);
                    acc[i][t] = th_mfma<FMT>(pl[i], bt[0], acc[i][t]);
                    if constexpr (NP == 2) acc[i][t] = th_mfma<FMT>(ph[i], bt[1], acc[i][t]);
                }
            }
        }
        if constexpr (Ring == 1) {
            if (c + 1 < nch) {
                lds_barrier();  // every wave is done with the chunk
                stage(c + 1);
                if (c + 2 < nch) fetch(c + 2);
                lds_barrier();
            }
        }
    }
    // ---- partials of the tile's nodes
    l_run += dpp_f32<0xB1>(l_run);
    l_run += dpp_f32<0x4E>(l_run);
    l_run += dpp_f32<0x141>(l_run);
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        if (i >= live) break;
        float *P = a.part + (size_t)(s.part0 + (first + i) * (s.ns + 1) + split) * 16 * 514;
#pragma unroll
        for (int t = 0; t < NC; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) P[(4 * g + e) * 512 + 16 * (NC * w + t) + n] = acc[i][t][e];
    }
    if ((tid & 7) == 0 && sq / 16 < live) {
        float *P = a.part + (size_t)(s.part0 + (first + sq / 16) * (s.ns + 1) + split) * 16 * 514 + 8192;
        P[sq % 16] = m_run;
        P[16 + sq % 16] = l_run;
    }
}

// Splits of the history: as many rows per split (a multiple of the chunk, at least kThMin) as it takes for
// the launch's workgroups, ceil(count / nm) per split, to be one round on the CUs.
constexpr int kThMin = 64;
int plan_tree(int fmt, const Dims &d, TreeTable &t, int ncu) {
    const bool kimi = d.NH == 16 && d.R == 512 && d.DR == 64;
    int most = 0, longest = 0;
    for (int b = 0; b < t.n; ++b) {
        most = std::max(most, t.s[b].count);
        longest = std::max(longest, t.s[b].ctx);
    }
    t.nm = !kimi ? 0 : most > 2 || fmt == kFmtF32 ? 4 : 2;
    auto splits = [](long ctx, long r) { return (ctx + r - 1) / r; };
    long r = kThMin;
    if (t.nm) {
        const long places = (long)ncu * (t.nm == 2 ? 2 : 1);
        auto groups = [&](long rows) {
            long n = 0;
            for (int b = 0; b < t.n; ++b) n += (t.s[b].count + t.nm - 1) / t.nm * splits(t.s[b].ctx, rows);
            return n;
        };
        long lo = kThMin / kThCh, hi = std::max(lo, splits(longest, kThCh));
        while (lo < hi) {  // groups() does not increase with the rows
            const long mid = (lo + hi) / 2;
            if (groups(mid * kThCh) <= places) hi = mid;
            else lo = mid + 1;
        }
        // the combine takes at most kMaxSplits partials of a node
        r = std::max(lo * kThCh, (splits(longest, kMaxSplits - 1) + kThCh - 1) / kThCh * kThCh);
    }
    int part = 0, unit = 0;
    for (int b = 0; b < t.n; ++b) {
        TreeSeq &s = t.s[b];
        s.rps = (int)r;
        s.ns = t.nm ? (int)splits(s.ctx, r) : 0;
        s.tiles = t.nm ? (s.count + t.nm - 1) / t.nm : 0;
        s.part0 = part;
        s.unit0 = unit;
        part += s.count * (s.ns + 1);
        unit += s.ns;
    }
    return part;
}

template <int FMT>
static void tree_launch(hipStream_t st, const TreeArgs &a) {
    if (a.t.nm == 0) {
        hipLaunchKernelGGL(k_tree_generic<FMT>, dim3((unsigned)(a.t.nodes * a.d.NH)), dim3(256), 0, st, a);
        return;
    }
    hipLaunchKernelGGL(k_tree_path<FMT>, dim3((unsigned)a.t.nodes), dim3(512), 0, st, a);
    int most = 0;  // workgroups of the fullest XCD (tree_unit)
    for (int x = 0; x < 8; ++x) {
        int n = 0;
        for (int b = 0; b < a.t.n; ++b) {
            const int first = (x - a.t.s[b].unit0) & 7;
            if (a.t.s[b].ns > first) n += (a.t.s[b].ns - first + 7) / 8 * a.t.s[b].tiles;
        }
        most = std::max(most, n);
    }
    if (most == 0) return;  // no history
    const dim3 grid((unsigned)(8 * most));
    if constexpr (FMT != kFmtF32) {
        if (a.t.nm == 2) {
            hipLaunchKernelGGL((k_tree_hist<FMT, 2>), grid, dim3(256), 0, st, a);
            return;
        }
    }
    hipLaunchKernelGGL((k_tree_hist<FMT, 4>), grid, dim3(512), 0, st, a);
}

hipError_t launch_tree_attention(hipStream_t st, int fmt, const TreeTable &t, const Dims &d, const DecodeWork &w) {
    if (d.R > 256 * kTgCols || d.DR > 256 || t.n < 1 || t.nodes < 1 || t.nodes > kTreeNodes) return hipErrorInvalidValue;
    if (t.nm != 0 && (d.NH != 16 || d.R != 512 || d.DR != 64)) return hipErrorInvalidValue;
    if (t.nm != 0 && t.nm != 4 && (t.nm != 2 || fmt == kFmtF32)) return hipErrorInvalidValue;
    TreeArgs a;
    a.t = t;
    a.d = d;
    a.qf = w.qf;
    a.part = w.part;
    a.smscale = 1.0f / sqrtf((float)d.QD);
    if (fmt == kFmtQ8) tree_launch<kFmtQ8>(st, a);
    else if (fmt == kFmtF32) tree_launch<kFmtF32>(st, a);
    else if (fmt == kFmtBF16) tree_launch<kFmtBF16>(st, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

// ================================================================ rows =================

// Bytes [lo, hi) from src to dst, both with the alignment of lo to 16 (bases of hipMalloc and equal
// offsets): whole 16-byte words by all threads of the block, the ends byte by byte.
__device__ __forceinline__ void copy_range(uint8_t *dst, const uint8_t *src, size_t lo, size_t hi) {
    const size_t a = (lo + 15) & ~(size_t)15, b = hi & ~(size_t)15;
    const int tid = threadIdx.x, nt = blockDim.x;
    if (a >= b) {
        for (size_t i = lo + tid; i < hi; i += nt) dst[i] = src[i];
        return;
    }
    for (size_t i = a + 16 * (size_t)tid; i < b; i += 16 * (size_t)nt) *(v4i *)(dst + i) = *(const v4i *)(src + i);
    for (size_t i = lo + tid; i < a; i += nt) dst[i] = src[i];
    for (size_t i = b + tid; i < hi; i += nt) dst[i] = src[i];
}

constexpr size_t kForkChunk = 32768;  // bytes of an array one block copies

// Block (x, y): chunk x of pair y's arrays, which are cut at multiples of kForkChunk one after another.
__global__ __launch_bounds__(256) void k_fork(ForkTable t) {
    const ForkDesc &f = t.d[blockIdx.y];
    size_t c = blockIdx.x;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        if (t.e[k] == 0) continue;
        const size_t lo = (size_t)f.r0 * t.e[k], hi = (size_t)f.r1 * t.e[k], base = lo & ~(kForkChunk - 1);
        const size_t n = (hi - base + kForkChunk - 1) / kForkChunk;
        if (c < n) {
            const size_t x = base + c * kForkChunk;
            copy_range((uint8_t *)f.dst[k], (const uint8_t *)f.src[k], x > lo ? x : lo, x + kForkChunk < hi ? x + kForkChunk : hi);
            return;
        }
        c -= n;
    }
}

hipError_t launch_fork(hipStream_t st, const ForkTable &t) {
    if (t.n < 1 || t.n > kForkBatch) return hipErrorInvalidValue;
    size_t most = 0;
    for (int i = 0; i < t.n; ++i) {
        size_t n = 0;
        for (int k = 0; k < 3; ++k) {
            if (t.e[k] == 0) continue;
            const size_t lo = (size_t)t.d[i].r0 * t.e[k], hi = (size_t)t.d[i].r1 * t.e[k];
            n += (hi - (lo & ~(kForkChunk - 1)) + kForkChunk - 1) / kForkChunk;
        }
        most = std::max(most, n);
    }
    if (most < 1 || most > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_fork, dim3((unsigned)most, (unsigned)t.n), dim3(256), 0, st, t);
    return hipGetLastError();
}

// Moves one array's rows: a thread owns a column of `U`-wide words and takes the rows in ascending
// order, eight loads at a time. A row's destination start + i is not above its source
// start + path[i], and later sources lie above earlier destinations, so no row is overwritten
// before it has been read, and no other thread touches the column.
template <class U>
__device__ __forceinline__ void move_rows(void *p, int e, const AcceptDesc &d) {
    const int words = e / (int)sizeof(U);
    U *base = (U *)p + (size_t)d.start * words;
    for (int c = threadIdx.x; c < words; c += blockDim.x)
        for (int i = 0; i < d.n; i += 8) {
            U v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (i + q < d.n) v[q] = base[(size_t)d.path[i + q] * words + c];
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (i + q < d.n) base[(size_t)(i + q) * words + c] = v[q];
        }
}

// One block per state and array.
__global__ __launch_bounds__(256) void k_accept(AcceptTable t) {
    const AcceptDesc &d = t.d[blockIdx.x];
    const int e = t.e[blockIdx.y];
    void *p = d.p[blockIdx.y];
    if (e == 0) return;
    if (e % 16 == 0) move_rows<v4i>(p, e, d);
    else if (e % 4 == 0) move_rows<uint32_t>(p, e, d);
    else if (e % 2 == 0) move_rows<uint16_t>(p, e, d);
    else move_rows<uint8_t>(p, e, d);
}

hipError_t launch_accept(hipStream_t st, const AcceptTable &t) {
    if (t.n < 1 || t.n > kAcceptBatch) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_accept, dim3((unsigned)t.n, 3), dim3(256), 0, st, t);
    return hipGetLastError();
}

}  // namespace kvl
