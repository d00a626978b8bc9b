// Kernels of branching histories (include/kvl/mla_hip.h): the attention of a tree of drafted tokens
// over a latent history, copies of a state's rows, and the compaction of an accepted path's rows.
#include <hip/hip_runtime.h>

#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "mla_device.h"
#include "mla_internal.h"

namespace kvl {

// ================================================================ tree attention =======

// Node i of a tree over a history of n rows (row n + i is its own) attends rows 0 .. n - 1, the rows
// of its ancestors and its own, in one softmax per head:
//   s_j = (q_lat . lat_j + q_rope . key_j) / sqrt(QD),  mix = sum_j softmax(s)_j lat_j.
// Rows of other branches are never read for it, so nothing they hold (NaN, infinities) reaches it.

template <int FMT>
__device__ __forceinline__ float tree_lat(const TreeRows &s, size_t row, int R, int k) {
    if (FMT == kFmtQ8) return (float)((const int8_t *)s.a)[row * R + k] * ((const float *)s.b)[row];
    if (FMT == kFmtF32) return ((const float *)s.a)[row * R + k];
    return bf16_to_f32(((const uint16_t *)s.a)[row * R + k]);
}
template <int FMT>
__device__ __forceinline__ float tree_key(const TreeRows &s, size_t row, int DR, int k) {
    if (FMT == kFmtQ8) return bf16_to_f32(((const uint16_t *)s.c)[row * DR + k]);
    if (FMT == kFmtF32) return ((const float *)s.b)[row * DR + k];
    return bf16_to_f32(((const uint16_t *)s.b)[row * DR + k]);
}

struct TreeArgs {
    TreeTable t;
    const float *qf;
    float *part;
    float smscale;
};
struct TreeNodeArgs {
    TreeRowsTable t;
    TreeNodes nd;
    const float *qf;
    float *part;
    float smscale;
    int NH, R, DR;
};

constexpr int kTgRows = 256;  // rows taken at a time: a thread per row
constexpr int kTgCols = 4;    // latent columns per thread: R <= 1024

// Any dims: one workgroup per (node, head) goes over the node's rows kTgRows at a time with the
// running maximum and sum of the softmax; a thread per row forms the scores, a thread per latent
// column the mix. The route for every other set of dims, other head counts at R = 512, DR = 64 among them: nothing is
// shared between heads or nodes, and each thread reads a row of its own, so it is bound by the latency of those
// reads. The whole call of 8 nodes over 1000 / 8192 rows, BF16 (us): 8 heads 195 / 1423, 64 heads 292 / 1940; 16
// heads on the route below 40 / 54. (A single-token decode at 8 heads takes 4545 / 55700.)
template <int FMT>
__global__ __launch_bounds__(256) void k_tree_generic(TreeNodeArgs a) {
    __shared__ float q[1024 + 256];
    __shared__ float p[kTgRows];
    __shared__ float redm[4], reds[4];
    __shared__ int path[kTreeNodes];
    __shared__ int npath;
    const int tid = threadIdx.x, NH = a.NH, R = a.R, DR = a.DR;
    const int k = blockIdx.x / NH, h = blockIdx.x % NH;
    const TreeRows s = a.t.s[a.nd.seq[k]];
    for (int i = tid; i < R + DR; i += 256) q[i] = a.qf[((size_t)k * NH + h) * (R + DR) + i];
    if (tid == 0) {  // the node and its ancestors, in the order of their rows
        int n = 0;
        for (int i = k - s.node0; i >= 0; i = a.nd.parent[s.node0 + i]) ++n;
        npath = n;
        for (int i = k - s.node0; i >= 0; i = a.nd.parent[s.node0 + i]) path[--n] = i;
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
    float *P = a.part + (size_t)(s.part0 + k - s.node0) * NH * (R + 2);
#pragma unroll
    for (int c = 0; c < kTgCols; ++c)
        if (tid + 256 * c < R) P[(size_t)h * R + tid + 256 * c] = acc[c];
    if (tid == 0) {
        P[(size_t)NH * R + h] = m;
        P[(size_t)NH * R + NH + h] = l;
    }
}

// ---- the history (Kimi shapes) ------------------------------------------------------------------

// A workgroup takes NM nodes of one tree (16 NM queries) over one split of the history, in chunks of 32
// rows (FP32: 16) that all its waves share in LDS: 2 NM waves,
//   scores: wave (m, kh) = node m's 16 heads x the rows over half kh of the 576 columns, the queries held
//     in registers; the two halves are added through LDS;
//   softmax: 8 threads per query, 4 rows (FP32: 2) each, running maximum (moved only when a chunk exceeds it by
//     more than ln 64, so that the sums are rarely scaled) and sum in registers; weights to LDS as the next
//     product's operand;
//   mix: every wave 512 / (2 NM) latent columns of all 16 NM queries, the rows read transposed.
// Operands are 16 bits wide, sums 32: the 32-bit query and weight enter as hi + lo (two products), the
// BF16 rows as they are, the FP32 rows as hi + lo too (without lo . lo: three products), all in bf16 (what
// is left out is below 2^-17 of an operand).
// Q8: the scores are int8 products of the codes as stored and the query as a whole number below 2^22 (a power of
// two times it) in three bytes, exact but for that rounding; a row's scale and the query's power multiply the
// sum. The mix takes the codes as fp16 (exact) and the weights in two fp16 parts; a row's scale multiplies its
// weight. To keep the weights within fp16 whatever the scales, the running maximum is that of score + the scale's
// exponent (in units of log2); the reference lies kThLow below it, so that weight times scale stays below 2^15 and
// fp16's smallest step, 2^-24, is 2^-30 of the largest weight. Both parts round to nearest: where one row outweighs
// many small ones, a loss that is always downward adds up over them, and the lo parts of the small ones, which a
// matrix instruction drops (it adds at most eight rows at a time) beside a sum 2^25 times theirs, are as often negative. Eight trees,
// one row of about 0.6 of the weight, latents with a common mean: an output of 32768 / 131072 rows (a quarter of them a
// split) is off by 3.5e-6 / 3.3e-6; parts cut toward zero 9e-6 / 2.9e-5, with the reference at the maximum too 1.6e-4 /
// 5.8e-4. An exponent below -84 counts as -84 there: over kThMax rows of scale zero the sum of the weights stays below
// 2^(15 + 84 + 19), and 2^9 splits of them can still be added.
// What bounds it: the issue of matrix and vector instructions beside each other. 64 nodes x 32768 Q8 rows: 144 us,
// 1.04 PFLOP/s of operand products of 16 bits' worth (two per product of the formula) where the library's large
// bf16 product reaches 1.19; 129 us with rows of zeros, whose products draw less power. A launch of one chunk a
// workgroup (table, queries, chunk, the passes that fill the pipe) takes 8 to 10 us with NM = 2, 12 to 16 with NM = 4.
constexpr int kThCh = 32;  // rows of a chunk (FP32: of two)
// Q8: the reference of the weights lies kThLow below the maximum that moves it (rounded: at most 8, whatever the size of
// the logits), which a later maximum may pass by kThTop.
constexpr float kThLow = 7.0f, kThTop = 15.0f;
template <int FMT, int NM>
struct ThShape {
    static constexpr int NW = 2 * NM, NT = 64 * NW, NQ = 16 * NM;
    static constexpr int NP = FMT == kFmtF32 ? 2 : 1;  // planes of a row
    static constexpr int Ch = kThCh / NP;              // rows of a chunk
    static constexpr bool Dma = FMT == kFmtQ8;         // rows go to LDS as they are stored
    static constexpr int RowB = FMT == kFmtQ8 ? 512 : 1024;
    static constexpr int LatB = Ch * RowB, KeyB = Ch * 128, PlaneB = LatB + KeyB;
    static constexpr int ScB = FMT == kFmtQ8 ? Ch * 4 : 0;  // scales
    static constexpr int Slot = NP * PlaneB + ScB;
    static constexpr bool Pipe = NM == 4;
    static constexpr int Ring = Pipe ? (Dma ? 5 : 3) : (Dma ? 2 : 1);
    static constexpr int SpOff = Ring * Slot;
    static constexpr int SpH = NQ * 36;  // floats of a half of the scores (th_sp)
    static constexpr int SpB = 2 * SpH * 4;
    static constexpr int PwOff = SpOff + (Pipe ? 2 : 1) * SpB;
    static constexpr int PwB = NQ * 64;  // bytes of a plane of weights (th_pw)
    static constexpr int PwN = Pipe && Dma ? 2 : 1;  // buffers of weights
    static constexpr int AlOff = PwOff + PwN * 2 * PwB;
    static constexpr int FlOff = AlOff + PwN * NQ * 4;
    static constexpr int Smem = FlOff + 2 * 8 * 4;
    static_assert(Smem <= 160 * 1024, "LDS of one CU");
};
// Places in LDS, chosen so that the lanes served together hit distinct banks. A 16-byte read serves 16
// lanes a cycle, and not neighbours: lanes 0-3, 12-15, 20-23, 24-27, then 4-7, 8-11, 16-19, 28-31 and so
// on (found with patterns of conflicting addresses and the LDS counters). With rows n = lane % 16 and
// words + lane / 16, as the products read, that is rows 0-3 and 12-15 of one word beside 4-11 of the next.
//   word c of latent row r: c ^ th_swz(r) (Q8, 512 bytes a row: c ^ (r & 15)), which also spreads the
//     transposed reads (4 rows x 32 bytes; Q8 16 rows x 16 bytes);
//   word of 8 weights of query q: th_pw;  score of query q, row 0 (floats): th_sp;
// 18 + 8 such reads of a chunk and wave, BF16: 97 -> 0 cycles of conflicts.
__device__ __forceinline__ int th_swz(int r) { return ((r & 3) << 1) | ((((r >> 2) ^ (r >> 3)) & 1) << 3) | ((r >> 3) & 1); }
__device__ __forceinline__ int th_sp(int q) { return (q >> 2) * 144 + (q & 3) * 32; }
__device__ __forceinline__ int th_pw(int q, int word) {
    const int z = (q >> 2) & 3;
    return q * 64 + 16 * (word ^ (((z ^ (z << 1)) & 2) | (z >> 1)));
}
// word c of key row r
__device__ __forceinline__ int th_key(int r, int c) { return r * 128 + 16 * (c ^ ((r >> 1) & 7)); }

// Workgroup -> (sequence, split, tile). The workgroups of a launch, sequence by sequence, split by split,
// the tiles of a split one after another, are cut into eight equal runs, one per XCD (workgroup i runs on
// XCD i % 8): an XCD's L2 serves the rows that the tiles of a split share, and no XCD has more workgroups
// than another. Lane b of every wave reads sequence b's entry; the workgroup's entry then comes from its
// lane, in scalar registers.
__device__ __forceinline__ int tree_lane(int v, int b) { return __builtin_amdgcn_readlane(v, b); }
__device__ __forceinline__ uint8_t *tree_lane(void *p, int b) {
    const uint64_t u = (uint64_t)p;
    const uint32_t lo = (uint32_t)tree_lane((int)(uint32_t)u, b), hi = (uint32_t)tree_lane((int)(uint32_t)(u >> 32), b);
    return (uint8_t *)(((uint64_t)hi << 32) | lo);
}
struct TreeUnit {
    uint8_t *a, *b, *c;
    int ctx, count, node0, part0, ns, rps, split, tile;
};
__device__ __forceinline__ bool tree_unit(const TreeTable &t, TreeUnit &u) {
    const int lane = threadIdx.x & 63, xcd = blockIdx.x & 7, j = blockIdx.x >> 3;
    const TreeSeq q = t.s[lane];
    const int each = t.units >> 3, more = t.units & 7;
    if (j >= each + (xcd < more ? 1 : 0)) return false;
    const int i = xcd * each + min(xcd, more) + j;
    const int b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane > 0 && lane < t.n && i >= q.unit0));
    const int r = i - tree_lane(q.unit0, b), tiles = tree_lane(q.tiles, b);
    u.split = r / tiles;
    u.tile = r % tiles;
    u.a = tree_lane(q.a, b);
    u.b = tree_lane(q.b, b);
    u.c = tree_lane(q.c, b);
    u.ctx = tree_lane(q.ctx, b);
    u.count = tree_lane(q.count, b);
    u.node0 = tree_lane(q.node0, b);
    u.part0 = tree_lane(q.part0, b);
    u.ns = tree_lane(q.ns, b);
    u.rps = tree_lane(q.rps, b);
    return true;
}

template <int FMT>
__device__ __forceinline__ v4f th_mfma(const v4i &a, const v4i &b, const v4f &c) {
    if (FMT == kFmtQ8) return mfma_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c);
    return mfma_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c);
}

// Eight fp32 values as hi and lo operands (bf16).
__device__ __forceinline__ void th_split(const v4f &x0, const v4f &x1, v4i &hi, v4i &lo) {
    v8bf h, r;
    split8_cvt(x0, x1, h, r);
    hi = __builtin_bit_cast(v4i, h);
    lo = __builtin_bit_cast(v4i, r);
}

// Eight int8 codes -> eight fp16 values, exact: the code + 128 as the low mantissa bits of 1024, minus
// 1152.
__device__ __forceinline__ v4i codes_f16(const v2i &c) {
    const v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t u = (uint32_t)c[i] ^ 0x80808080u;
        o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off);
        o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off);
    }
    return v4i{(int)o[0], (int)o[1], (int)o[2], (int)o[3]};
}

// Four weights as hi and lo halves, rounded to nearest: what is left out is at most 2^-17 of the weight (bf16) or 2^-23
// (fp16; 2^-25 absolute where that is more, below a weight of 1/4).
template <bool F16>
__device__ __forceinline__ void th_split4(const v4f &x, int2 &hi, int2 &lo) {
    if constexpr (F16) {
        const v2h h0 = __builtin_convertvector((v2f{x[0], x[1]}), v2h), h1 = __builtin_convertvector((v2f{x[2], x[3]}), v2h);
        const v2h l0 = __builtin_convertvector((v2f{x[0] - (float)h0.x, x[1] - (float)h0.y}), v2h);
        const v2h l1 = __builtin_convertvector((v2f{x[2] - (float)h1.x, x[3] - (float)h1.y}), v2h);
        hi = int2{__builtin_bit_cast(int, h0), __builtin_bit_cast(int, h1)};
        lo = int2{__builtin_bit_cast(int, l0), __builtin_bit_cast(int, l1)};
    } else {
        const v2bf h0 = __builtin_convertvector((v2f{x[0], x[1]}), v2bf), h1 = __builtin_convertvector((v2f{x[2], x[3]}), v2bf);
        const v2bf l0 = __builtin_convertvector((v2f{x[0] - (float)h0.x, x[1] - (float)h0.y}), v2bf);
        const v2bf l1 = __builtin_convertvector((v2f{x[2] - (float)h1.x, x[3] - (float)h1.y}), v2bf);
        hi = int2{__builtin_bit_cast(int, h0), __builtin_bit_cast(int, h1)};
        lo = int2{__builtin_bit_cast(int, l0), __builtin_bit_cast(int, l1)};
    }
}

template <int FMT, int NM>
__global__ __launch_bounds__(128 * NM) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_tree_hist(TreeArgs a) {
    using Sh = ThShape<FMT, NM>;
    constexpr int NT = Sh::NT, NW = Sh::NW, NP = Sh::NP, Ch = Sh::Ch, RB = Ch / 16;
    constexpr int NC = 512 / NW / 16;  // 16-column blocks of a wave in the mix
    constexpr bool kQ8 = FMT == kFmtQ8;
    __shared__ __attribute__((aligned(16))) uint8_t smem[Sh::Smem];
    const int tid = threadIdx.x, l = tid & 63, n = l & 15, g = l >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    TreeUnit s;
    if (!tree_unit(a.t, s)) return;
    const int split = s.split, tile = s.tile;
    const int r0 = split * s.rps, r1 = split == s.ns - 1 ? s.ctx : r0 + s.rps;
    const int nch = (r1 - r0 + Ch - 1) / Ch;
    const int first = tile * NM, live = min(NM, s.count - first);  // nodes of this tile

    // ---- Q8: a chunk's rows from memory to an LDS slot, asynchronously. One instruction of a wave takes 1 KB,
    // two rows of codes; the wave's keys and scales are one instruction each. Rows past the split repeat its
    // last one (their scores are masked).
    constexpr int KR = Ch / NW, NA = kQ8 ? Ch / 2 / NW : 0;  // a wave's key rows, pairs of rows of codes
    auto issue = [&](int c, int slot) __attribute__((always_inline)) {
        if constexpr (kQ8) {
            const int last = r1 - r0 - 1;
            const uint32_t to = lds_addr(smem) + slot * Sh::Slot;
            const int lr = 2 * w + (l >> 5), sw = 16 * ((l & 31) ^ (lr & 15));
#pragma unroll
            for (int i = 0; i < NA; ++i)  // row lr + 2 NW i
                dma_b128_s(s.a + (size_t)r0 * 512, (uint32_t)(min(c * Ch + lr + 2 * NW * i, last) * 512 + (sw ^ (16 * ((2 * NW * i) & 15)))),
                           to + (NW * i + w) * 1024);
            const int kr = KR * w + (l >> 3);
            if (l < 8 * KR)
                dma_b128_s(s.c + (size_t)r0 * 128, (uint32_t)(min(c * Ch + kr, last) * 128 + 16 * ((l & 7) ^ ((kr >> 1) & 7))),
                           to + Sh::LatB + 128 * KR * w);
            if (l < KR) dma_b32(s.b + 4 * ((size_t)r0 + min(c * Ch + KR * w + l, last)), to + Sh::PlaneB + 4 * KR * w);
        }
    };
    // ---- BF16, FP32: from memory to registers, and from there to an LDS slot. A thread
    // takes eight values of a latent row (word tid % 64 of rows tid / 64 + NW i) and eight bytes of a key row
    // (tid % 16 of rows tid / 16 + NT / 16 i; FP32: tid % 32 of rows tid / 32).
    constexpr int NL = Ch / NW, NK = 512 / NT;
    constexpr int LE = FMT == kFmtF32 ? 4 : 2, KE = LE;  // bytes of an element
    constexpr int LV = LE == 4 ? 2 : 1;
    struct Held {
        v4i la[NL * LV];
        v2i kb[NK];
    };
    const int lrow = tid >> 6;
    // the split's rows as buffers: a read past the last row gives zeros (its score is masked)
    const int nrow = r1 - r0;
    const auto ba = __builtin_amdgcn_make_buffer_rsrc(s.a + (size_t)r0 * (512 * LE), 0, nrow * (512 * LE), 0x00027000);
    const auto bk = __builtin_amdgcn_make_buffer_rsrc(s.b + (size_t)r0 * (64 * KE), 0, nrow * (64 * KE), 0x00027000);
    const int va = tid * (8 * LE), vk = tid * 8;  // rows lie one after another, so do the threads' words
    auto fetch = [&](int c, Held &f) __attribute__((always_inline)) {
        const int oa = va + c * (Ch * 512 * LE), ok = vk + c * (Ch * 64 * KE);
#pragma unroll
        for (int i = 0; i < NL; ++i)
#pragma unroll
            for (int v = 0; v < LV; ++v)
                f.la[LV * i + v] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(ba, oa + i * (NT * 8 * LE) + 16 * v, 0, 0));
#pragma unroll
        for (int i = 0; i < NK; ++i) f.kb[i] = __builtin_bit_cast(v2i, __builtin_amdgcn_raw_buffer_load_b64(bk, ok + i * (NT * 8), 0, 0));
    };
    auto put = [&](uint8_t *at, const v4i *v) __attribute__((always_inline)) {
        if constexpr (NP == 2) {
            v4i hi, lo;
            th_split(__builtin_bit_cast(v4f, v[0]), __builtin_bit_cast(v4f, v[1]), hi, lo);
            *(v4i *)at = hi;
            *(v4i *)(at + Sh::PlaneB) = lo;
        } else {
            *(v4i *)at = v[0];
        }
    };
    const int sa = lrow * 1024 + 16 * (l ^ th_swz(lrow));
    const int sk = Sh::LatB + (KE == 4 ? th_key(tid >> 5, (tid >> 2) & 7) + 4 * (tid & 3) : th_key(tid >> 4, (tid >> 1) & 7) + 8 * (tid & 1));
    // piece i < NL: a latent item; the last piece: the key items
    auto stage = [&](uint8_t *buf, const Held &f, int i) __attribute__((always_inline)) {
        if (i < NL) {
            // row lrow + NW i: th_swz changes by the bits of NW i below 16
            uint8_t *at = buf + (sa ^ (16 * th_swz((NW * i) & 15))) + NW * i * 1024;
            put(at, f.la + LV * i);
            return;
        }
#pragma unroll
        for (int q = 0; q < NK; ++q) {
            if constexpr (KE == 4) {
                const v2f x = __builtin_bit_cast(v2f, f.kb[q]);
                const v2bf hi = __builtin_convertvector(x, v2bf);
                const v2bf lo = __builtin_convertvector((v2f{x.x - (float)hi.x, x.y - (float)hi.y}), v2bf);
                const int at = (sk ^ (64 * q)) + q * 1024;  // 8 rows on (four waves): th_key flips one bit of the word
                *(int *)(buf + at) = __builtin_bit_cast(int, hi);
                *(int *)(buf + Sh::PlaneB + at) = __builtin_bit_cast(int, lo);
            } else {
                *(v2i *)(buf + sk + q * (NT / 16) * 128) = f.kb[q];
            }
        }
    };
    auto stage_all = [&](uint8_t *buf, const Held &f) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i <= NL; ++i) stage(buf, f, i);
    };

    Held held, ahead;  // the first two chunks are requested together
    if constexpr (Sh::Dma) {
        issue(0, 0);
    } else {
        fetch(0, ahead);
        fetch(1, held);
    }
    // ---- queries: A operand of the scores, head n of node m: columns 32 kb + 8 g .. of the eight
    // latent blocks kb = 8 kh + j and of the key block kh (the last). Q8: columns 64 kb + 16 g .. of the four blocks
    // kb = 4 kh + j as whole numbers below 2^22 in three signed bytes, qp[3 j] the high one. Scores are in
    // units of log2.
    const int m = w % NM, kh = w / NM;
    constexpr int NQK = kQ8 ? 1 : 9;
    v4i qh[NQK], ql[NQK], qp[kQ8 ? 12 : 1];
    float qd[4] = {1.f, 1.f, 1.f, 1.f};  // Q8: undoes the query's power of two, heads 4 g + i
    {
        const float *qrow = a.qf + ((size_t)(s.node0 + first + min(m, live - 1)) * 16 + n) * 576;
        const float unit = a.smscale * 1.44269504f;
        v4f qv[18];
#pragma unroll
        for (int j = 0; j < 9; ++j) {
            const int col = j == 8 ? 512 + 32 * kh + 8 * g
                            : kQ8  ? 256 * kh + 64 * (j >> 1) + 16 * g + 8 * (j & 1)
                                   : 32 * (8 * kh + j) + 8 * g;
            const float *p = qrow + col;
            qv[2 * j] = *(const v4f *)p * unit;
            qv[2 * j + 1] = *(const v4f *)(p + 4) * unit;
        }
        if constexpr (kQ8) {
            float mx = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(qv[j][e]));
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            // 2^(22 - e) with 2^(e - 1) <= mx < 2^e, from the exponent's bits, at most 2^104. (A query that is not
            // finite is cut here: the node's own row, which it attends, makes its output NaN.)
            const int e = max((int)((__float_as_uint(mx) >> 23) & 255) - 126, -82);
            const float qs = __uint_as_float((uint32_t)(149 - e) << 23);
            const float qi = __uint_as_float((uint32_t)(105 + e) << 23);
#pragma unroll
            for (int i = 0; i < 4; ++i) qd[i] = __shfl(qi, 4 * g + i);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    uint32_t b0 = 0, b1 = 0, b2 = 0;
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int v = (int)rintf(__builtin_amdgcn_fmed3f(qv[4 * j + z][y] * qs, -4194304.f, 4194304.f));
                        const int v1 = (v + 128) >> 8, v0 = (v1 + 128) >> 8;  // v - 256 v1, v1 - 256 v0: a signed byte each
                        b0 |= (uint32_t)(v0 & 255) << (8 * y);
                        b1 |= (uint32_t)(v1 & 255) << (8 * y);
                        b2 |= (uint32_t)(v & 255) << (8 * y);
                    }
                    qp[3 * j][z] = (int)b0;
                    qp[3 * j + 1][z] = (int)b1;
                    qp[3 * j + 2][z] = (int)b2;
                }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) th_split(qv[2 * j], qv[2 * j + 1], qh[j], ql[j]);
        }
        th_split(qv[16], qv[17], qh[NQK - 1], ql[NQK - 1]);
    }
    if constexpr (!Sh::Dma) stage_all(smem, ahead);

    // score operands: row n of a 16-row half, block j at bofs[j % 4] + 256 (j / 4) (Q8: bofs[j])
    int bofs[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        bofs[j] = n * Sh::RowB + 16 * (kQ8 ? (4 * (4 * kh + j) + g) ^ n : (4 * (8 * kh + j) + g) ^ th_swz(n));
    const int kofs = Sh::LatB + th_key(n, 4 * kh + g);
    // transposed reads of column block NC w + t (lds_read_tr16): rows 8 g + 4 h + (n >> 2); of the FP32 planes
    // the 16 hi rows for g = 0, 1 and the 16 lo rows for g = 2, 3
    // Q8 (lds_read_tr8): rows 8 g + (n >> 1), 16 columns a word, read t at tro[0][0] ^ 16 t.
    int tro[2][NC];
    if constexpr (kQ8) {
        const int row = 8 * g + (n >> 1);
        tro[0][0] = row * 512 + 16 * ((NC * w) ^ (row & 15)) + 8 * (n & 1);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = 8 * (NP == 2 ? g & 1 : g) + 4 * h + (n >> 2);
#pragma unroll
            for (int t = 0; t < NC; ++t)
                tro[h][t] = (NP == 2 ? (g >> 1) * Sh::PlaneB : 0) + row * 1024 +
                            16 * ((2 * (NC * w + t) + ((n >> 1) & 1)) ^ th_swz(row)) + 8 * (n & 1);
        }
    }
    constexpr int SR = Ch / 8;                      // softmax: rows of a thread,
    const int sq = tid >> 3, sr = SR * (tid & 7);  // its query and first row
    float m_run = -3e38f, l_run = 0.f;  // below any score but those at fp32's end (-inf would make its own rows' weights NaN)
    v4f acc[NM][NC];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int t = 0; t < NC; ++t) acc[i][t] = v4f{0.f, 0.f, 0.f, 0.f};
    lds_barrier();

    // The operand reads of a product run W reads ahead of it. The order below is kept as it is written: left
    // to itself the compiler reads each operand right before its use and waits for LDS every time.
    const int spw = Sh::SpOff + 4 * (kh * Sh::SpH + th_sp(16 * m + 4 * g) + n), spr = Sh::SpOff + 4 * (th_sp(sq) + sr);
    // the sums of a query's three bytes together (256 b + c: below 2^31)
    auto whole = [](int a, int b, int c) __attribute__((always_inline)) { return fmaf((float)a, 65536.f, (float)(256 * b + c)); };
    // between(i): other work after read i's products
    auto scores_q8 = [&](const uint8_t *buf, int c, auto between) __attribute__((always_inline)) {
        float *sp = (float *)(smem + spw + (Sh::Pipe ? (c & 1) * Sh::SpB : 0));
        // read i: block i / RB of rows 16 (i % RB); the last RB reads: the keys
        constexpr int N = 5 * RB, W = 6;
        auto get = [&](int i) __attribute__((always_inline)) {
            const int j = i / RB, rb = i % RB;
            return *(const v4i *)(buf + (j < 4 ? bofs[j] + 8192 * rb : kofs + 2048 * rb));
        };
        v4i d[3][RB], bv[W];  // by the bytes of the query
        v4f dk[RB];
        float x[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            dk[rb] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int z = 0; z < 3; ++z) d[z][rb] = v4i{0, 0, 0, 0};
            x[rb] = *(const float *)(buf + Sh::PlaneB + 4 * (16 * rb + n));
        }
#pragma unroll
        for (int i = 0; i < W; ++i) bv[i] = get(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = i / RB, rb = i % RB;
            const v4i v = bv[i % W];
            if (j < 4) {
#pragma unroll
                for (int z = 0; z < 3; ++z) d[z][rb] = mfma_i8(qp[kQ8 ? 3 * j + z : 0], v, d[z][rb]);
            } else {
                dk[rb] = th_mfma<kFmtBF16>(qh[0], v, dk[rb]);
                dk[rb] = th_mfma<kFmtBF16>(ql[0], v, dk[rb]);
            }
            if (i + W < N) bv[i % W] = get(i + W);
            between(i);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sp[32 * i + 16 * rb] = fmaf(whole(d[0][rb][i], d[1][rb][i], d[2][rb][i]), qd[i] * x[rb], dk[rb][i]);
            }
    };
    auto scores = [&](const uint8_t *buf, int c, auto between) __attribute__((always_inline)) {
        if constexpr (kQ8) {
            scores_q8(buf, c, between);
            return;
        }
        float *sp = (float *)(smem + spw + (Sh::Pipe ? (c & 1) * Sh::SpB : 0));
        // read i: plane i % NP of rows 16 (i / NP % RB) of block i / NP / RB
        constexpr int N = 9 * NP * RB, W = 6;
        auto get = [&](int i) __attribute__((always_inline)) {
            const int j = i / (NP * RB), rb = i / NP % RB;
            return *(const v4i *)(buf + (i % NP) * Sh::PlaneB + (j < 8 ? bofs[j & 3] + 256 * (j >> 2) + 16384 * rb : kofs + 2048 * rb));
        };
        // sums: d over the latents by rows (FP32: by hi . hi and lo . hi), dk over the key (FP32: hi . lo)
        v4f d[2], dk;
        v4i bv[W];
#pragma unroll
        for (int z = 0; z < 2; ++z) d[z] = dk = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < W; ++i) bv[i] = get(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = i / (NP * RB) % NQK, rb = i / NP % RB;
            const v4i v = bv[i % W];
            if constexpr (NP == 2) {  // not lo . lo
                if (i % 2 == 0) {
                    d[0] = th_mfma<FMT>(qh[j], v, d[0]);
                    d[1] = th_mfma<FMT>(ql[j], v, d[1]);
                } else {
                    dk = th_mfma<FMT>(qh[j], v, dk);
                }
            } else {
                d[rb] = th_mfma<FMT>(qh[j], v, d[rb]);
                d[rb] = th_mfma<FMT>(ql[j], v, d[rb]);
            }
            if (i + W < N) bv[i % W] = get(i + W);
            between(i);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (NP == 2) d[0] += d[1] + dk;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int i = 0; i < 4; ++i) sp[32 * i + 16 * rb] = d[rb][i];
    };
    // softmax of a chunk: its reads, then its arithmetic and writes in five pieces
    typedef float vsr __attribute__((ext_vector_type(SR)));
    vsr sx, sr4, sp4;
    float cm, alpha;
    bool moved;
    auto softmax_read = [&](const uint8_t *buf, int c) __attribute__((always_inline)) {
        const float *sp = (const float *)(smem + spr + (Sh::Pipe ? (c & 1) * Sh::SpB : 0));
        const vsr s0 = *(const vsr *)sp, s1 = *(const vsr *)(sp + Sh::SpH);
        if constexpr (kQ8) sr4 = *(const vsr *)(buf + Sh::PlaneB + 4 * sr);
        sx = s0 + s1;
    };
    auto softmax = [&](int c, int piece) __attribute__((always_inline)) {
        if (piece == 0) {
            // of a chunk's rows, the ones in the split; none before the first chunk
            const int rows = c < 0 ? 0 : r1 - (r0 + c * Ch);
            if (rows < Ch)
#pragma unroll
                for (int e = 0; e < SR; ++e) sx[e] = sr + e < rows ? sx[e] : -INFINITY;
            vsr t = sx;
            if constexpr (kQ8)
#pragma unroll
                for (int e = 0; e < SR; ++e) t[e] += (float)max(__builtin_amdgcn_frexp_expf(sr4[e]), -84);
            cm = fmaxf(t[0], t[1]);
            if constexpr (SR == 4) cm = fmaxf(cm, fmaxf(t[2], t[3]));
            cm = fmaxf(cm, dpp_f32<0xB1>(cm));
        } else if (piece == 1) {
            cm = fmaxf(cm, dpp_f32<0x4E>(cm));
            cm = fmaxf(cm, dpp_f32<0x141>(cm));  // row_half_mirror: the other four of the eight
            // as differences, exact where they decide: of logits past 2^24 sums would round by more than 1
            const bool mv = cm - m_run > (kQ8 ? kThTop : 6.0f);
            const float to = kQ8 ? cm - kThLow : cm;
            moved = __any(mv);
            alpha = mv ? __builtin_amdgcn_exp2f(m_run - to) : 1.0f;
            m_run = mv ? to : m_run;
        } else if (piece == 2) {
#pragma unroll
            for (int e = 0; e < SR; ++e) sp4[e] = __builtin_amdgcn_exp2f(sx[e] - m_run);
        } else if (piece == 3) {
            // this thread's rows; the eight threads' sums are added at the end
            float sum = sp4[0] + sp4[1];
            if constexpr (SR == 4) sum += sp4[2] + sp4[3];
            l_run = fmaf(l_run, alpha, sum);
            if constexpr (kQ8) sp4 *= sr4;
        } else {
            if constexpr (SR == 4) {
                int2 hi, lo;
                th_split4<kQ8>(sp4, hi, lo);
                uint8_t *pw = smem + Sh::PwOff + (Sh::PwN == 2 ? (c & 1) * 2 * Sh::PwB : 0) + th_pw(sq, sr >> 3) + 2 * (sr & 4);
                *(int2 *)pw = hi;
                *(int2 *)(pw + Sh::PwB) = lo;
            } else {  // the hi weights in words 0, 1, the lo weights in words 2, 3
                const v2bf hi = __builtin_convertvector((v2f{sp4[0], sp4[1]}), v2bf);
                const v2bf lo = __builtin_convertvector((v2f{sp4[0] - (float)hi.x, sp4[1] - (float)hi.y}), v2bf);
                *(int *)(smem + Sh::PwOff + th_pw(sq, sr >> 3) + 2 * (sr & 7)) = __builtin_bit_cast(int, hi);
                *(int *)(smem + Sh::PwOff + th_pw(sq, 2 + (sr >> 3)) + 2 * (sr & 7)) = __builtin_bit_cast(int, lo);
            }
            if ((tid & 7) == 0) *(float *)(smem + Sh::AlOff + (Sh::PwN == 2 ? (c & 1) * 4 * Sh::NQ : 0) + 4 * sq) = alpha;
            if (l == 0) *(int *)(smem + Sh::FlOff + 32 * (c & 1) + 4 * w) = moved ? 1 : 0;
        }
    };
    auto mix = [&](const uint8_t *buf, int c, auto between) __attribute__((always_inline)) {
        // FP32: an operand holds 16 rows twice, for the hi and for the lo plane: ph . (hi | lo) + pl . (hi | lo)
        v4i f[NW / 4], ph[NM], pl[NM], bt[2];
        v2i raw;  // Q8: the codes of the read after next
#pragma unroll
        for (int i = 0; i < NW / 4; ++i) f[i] = *(const v4i *)(smem + Sh::FlOff + 32 * (c & 1) + 16 * i);
        auto get = [&](int t) __attribute__((always_inline)) {
            if constexpr (kQ8)
                raw = lds_read_tr8(buf + (tro[0][0] ^ (16 * t)));
            else
                bt[t & 1] = __builtin_bit_cast(
                v4i, __builtin_shufflevector(lds_read_tr16(buf + tro[0][t]), lds_read_tr16(buf + tro[1][t]), 0, 1, 2, 3, 4, 5, 6, 7));
        };
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            ph[i] = *(const v4i *)(smem + Sh::PwOff + th_pw(16 * i + n, NP == 2 ? g & 1 : g));
            if (i == 0) get(0);
            pl[i] = *(const v4i *)(smem + Sh::PwOff + (NP == 2 ? th_pw(16 * i + n, 2 + (g & 1)) : Sh::PwB + th_pw(16 * i + n, g)));
        }
        if constexpr (kQ8) bt[0] = codes_f16(raw);
        get(1);
        int any = 0;
#pragma unroll
        for (int i = 0; i < NW / 4; ++i) any |= f[i][0] | f[i][1] | f[i][2] | f[i][3];
        if (__builtin_amdgcn_readfirstlane(any)) {
#pragma unroll
            for (int i = 0; i < NM; ++i) {
                const v4f al = *(const v4f *)(smem + Sh::AlOff + 64 * i + 16 * g);
#pragma unroll
                for (int t = 0; t < NC; ++t) acc[i][t] *= al;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < NC; ++t) {
#pragma unroll
            for (int i = 0; i < NM; ++i) acc[i][t] = th_mfma<FMT>(ph[i], bt[t & 1], acc[i][t]);
#pragma unroll
            for (int i = 0; i < NM; ++i) acc[i][t] = th_mfma<FMT>(pl[i], bt[t & 1], acc[i][t]);
            if constexpr (kQ8) bt[(t + 1) & 1] = codes_f16(raw);
            if (t + 2 < NC) get(t + 2);
            between(t);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // A pass of the Q8 pipe: scores of chunk c + 2, softmax of chunk c + 1, mix of chunk c. None needs another's
    // results, so a pass is one stream of products with the rest laid between them, and one barrier. The first
    // operands of the scores of chunk c + 3 are read at its end: the products start right behind the barrier.
    constexpr int W = 6;
    v4i bv[W];
    float bx[RB];
    auto first_reads = [&](const uint8_t *b, int i) __attribute__((always_inline)) {
        bv[i] = *(const v4i *)(b + bofs[i / RB] + 8192 * (i % RB));
        if (i < RB) bx[i] = *(const float *)(b + Sh::PlaneB + 4 * (16 * i + n));
    };
    auto pass = [&](int c, const uint8_t *b0, const uint8_t *b1, const uint8_t *b2, const uint8_t *b3) __attribute__((always_inline)) {
        constexpr int N = 5 * RB;  // as scores_q8
        float *sp = (float *)(smem + spw + (c & 1) * Sh::SpB);
        const uint8_t *pw = smem + Sh::PwOff + (c & 1) * 2 * Sh::PwB;
        auto get = [&](int i) __attribute__((always_inline)) {
            const int j = i / RB, rb = i % RB;
            return *(const v4i *)(b2 + (j < 4 ? bofs[j] + 8192 * rb : kofs + 2048 * rb));
        };
        auto codes = [&](int t) __attribute__((always_inline)) { return lds_read_tr8(b0 + (tro[0][0] ^ (16 * t))); };
        v4i d[3][RB], f[NW / 4], ph[NM], pl[NM], bt[2];
        v4f dk[RB];
        v2i raw[2];
        float x[RB];
        softmax_read(b1, c + 1);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            dk[rb] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int z = 0; z < 3; ++z) d[z][rb] = v4i{0, 0, 0, 0};
            x[rb] = bx[rb];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = i / RB, rb = i % RB;
            const v4i v = bv[i % W];
            if (j < 4) {
#pragma unroll
                for (int z = 0; z < 3; ++z) d[z][rb] = mfma_i8(qp[kQ8 ? 3 * j + z : 0], v, d[z][rb]);
            } else {
                dk[rb] = th_mfma<kFmtBF16>(qh[0], v, dk[rb]);
                dk[rb] = th_mfma<kFmtBF16>(ql[0], v, dk[rb]);
            }
            if (i + W < N) bv[i % W] = get(i + W);
            else if (i - (N - W) < NM) {  // the mix's operands
                const int k = i - (N - W);
                ph[k] = *(const v4i *)(pw + th_pw(16 * k + n, g));
                pl[k] = *(const v4i *)(pw + Sh::PwB + th_pw(16 * k + n, g));
                if (k < 2) raw[k] = codes(k);
                if (k < NW / 4) f[k] = *(const v4i *)(smem + Sh::FlOff + 32 * (c & 1) + 16 * k);
            }
            if (i >= 1 && i <= 5) softmax(c + 1, i - 1);
            if (i == N - 2) bt[0] = codes_f16(raw[0]);
            __builtin_amdgcn_sched_barrier(0);
        }
        int any = 0;
#pragma unroll
        for (int i = 0; i < NW / 4; ++i) any |= f[i][0] | f[i][1] | f[i][2] | f[i][3];
        if (__builtin_amdgcn_readfirstlane(any)) {
#pragma unroll
            for (int i = 0; i < NM; ++i) {
                const v4f al = *(const v4f *)(smem + Sh::AlOff + (c & 1) * 4 * Sh::NQ + 64 * i + 16 * g);
#pragma unroll
                for (int t = 0; t < NC; ++t) acc[i][t] *= al;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < NC; ++t) {
#pragma unroll
            for (int i = 0; i < NM; ++i) acc[i][t] = th_mfma<FMT>(ph[i], bt[t & 1], acc[i][t]);
#pragma unroll
            for (int i = 0; i < NM; ++i) acc[i][t] = th_mfma<FMT>(pl[i], bt[t & 1], acc[i][t]);
            if (t + 1 < NC) bt[(t + 1) & 1] = codes_f16(raw[(t + 1) & 1]);
            if (t + 2 < NC) raw[t & 1] = codes(t + 2);
            if (t < RB)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sp[32 * i + 16 * t] = fmaf(whole(d[0][t][i], d[1][t][i], d[2][t][i]), qd[i] * x[t], dk[t][i]);
            else
#pragma unroll
                for (int i = 3 * (t - RB); i < 3 * (t - RB) + 3; ++i) first_reads(b3, i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NM; ++i)
#pragma unroll
            for (int t = 0; t < NC; ++t) acc[i][t] = v4f{0.f, 0.f, 0.f, 0.f};
    };

    if constexpr (Sh::Pipe && Sh::Dma) {
        // Five slots: chunks c .. c + 3 in use, c + 4 on its way. The passes c = -2, -1 fill the pipe (the softmax of
        // a chunk below 0 has no rows, the sums are dropped); what the last passes bring and score is not used.
        auto slot = [&](int k) __attribute__((always_inline)) { return smem + k * Sh::Slot; };
        issue(1, 1);
        wait_vmcnt<0>();
        lds_barrier();
#pragma unroll
        for (int i = 0; i < W; ++i) first_reads(slot(0), i);
        int k0 = 3, k1 = 4, k2 = 0, k3 = 1, k4 = 2;  // slots of chunks c .. c + 4
        for (int c = -2; c < nch; ++c) {
            issue(c + 4, k4);  // its slot was chunk c - 1's
            pass(c, slot(k0), slot(k1), slot(k2), slot(k3));
            if (c < 0) clear();
            wait_vmcnt<0>();  // chunk c + 4 has come
            lds_barrier();
            const int t = k0;
            k0 = k1;
            k1 = k2;
            k2 = k3;
            k3 = k4;
            k4 = t;
        }
    } else if constexpr (Sh::Pipe) {
        // Two barriers a chunk. Between them a wave holds a product and vector work that do not depend on each
        // other, the vector work laid between the products: scores of chunk c + 1 with the softmax of chunk
        // c, then the mix of chunk c with the staging of chunk c + 2. The pass c = -1 fills the pipe (its
        // softmax has no rows, its sums are dropped); what the last passes stage and score is not used.
        static_assert(NL <= NC, "a latent item per column block");
        uint8_t *cur = smem + 2 * Sh::Slot, *next = smem, *then = smem + Sh::Slot;
        for (int c = -1; c < nch; ++c) {
            softmax_read(cur, c);
            scores(next, c + 1, [&](int i) __attribute__((always_inline)) {
                if (i >= 4 && i <= 12 && i % 2 == 0) softmax(c, (i - 4) / 2);
            });
            lds_barrier();
            mix(cur, c, [&](int t) __attribute__((always_inline)) {
                if (t < NL) stage(then, held, t);
                if (t == NC - 1) stage(then, held, NL);
            });
            fetch(c + 3, held);
            if (c < 0) clear();
            lds_barrier();
            uint8_t *t = cur;
            cur = next;
            next = then;
            then = t;
        }
    } else if constexpr (Sh::Dma) {
        wait_vmcnt<0>();
        lds_barrier();
        for (int c = 0; c < nch; ++c) {
            const uint8_t *buf = smem + (c & 1) * Sh::Slot;
            if (c + 1 < nch) issue(c + 1, (c + 1) & 1);
            scores(buf, c, [](int) {});
            lds_barrier();  // both halves of every score are in LDS
            softmax_read(buf, c);
#pragma unroll
            for (int i = 0; i < 5; ++i) softmax(c, i);
            lds_barrier();  // the weights are in LDS
            mix(buf, c, [](int) {});
            wait_vmcnt<0>();  // the next chunk has come
            lds_barrier();
        }
    } else {
        for (int c = 0; c < nch; ++c) {
            scores(smem, c, [](int) {});
            lds_barrier();  // both halves of every score are in LDS
            softmax_read(smem, c);
#pragma unroll
            for (int i = 0; i < 5; ++i) softmax(c, i);
            lds_barrier();  // the weights are in LDS
            mix(smem, c, [](int) {});
            if (c + 1 < nch) {
                lds_barrier();  // every wave is done with the chunk
                stage_all(smem, held);
                fetch(c + 2, held);
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
        float *P = a.part + (size_t)(s.part0 + (first + i) * s.ns + split) * 16 * 514;
#pragma unroll
        for (int t = 0; t < NC; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) P[(4 * g + e) * 512 + 16 * (NC * w + t) + n] = acc[i][t][e];
    }
    if ((tid & 7) == 0 && sq / 16 < live) {
        float *P = a.part + (size_t)(s.part0 + (first + sq / 16) * s.ns + split) * 16 * 514 + 8192;
        P[sq % 16] = m_run * 0.693147181f;  // in units of the natural logarithm
        P[16 + sq % 16] = l_run;
    }
}

// ---- the nodes' own rows, the merge and W_UV (Kimi shapes, DV = 128) --------------------------------

constexpr int kTcAhead = 6;  // splits whose loads a wave has in flight
struct TreeCombArgs {
    TreeRowsTable t;
    TreeNodes nd;
    const float *qf, *part;
    const uint16_t *kv_b;
    uint16_t *hos;
    size_t plane;  // words between the hi and lo planes of hos
    float smscale;
    int DN, n, tn;  // n nodes, tn of them per workgroup (EARLY: 1, 2, 4; else 8)
};

// Workgroup = one head of tn nodes, eight waves, 8 / tn of them per node (in turn over the history's splits).
// Bound by latency: table -> path -> partials -> W_UV, 8.5 us for a few nodes of a short history, 16 us at 4 nodes x 256
// splits, 22 us at 256 nodes x 4 splits (34 MB of partials, 67 MB of W_UV from L2).
//   merge: mix = (sum_s e^(m_s - M) acc_s + the path's) / (sum_s e^(m_s - M) l_s + the path's), lane l columns
//     4 l .. and 256 + 4 l ..;
//   path: the node's first wave takes the node's own row and its ancestors' (rows ctx + i, at most 64), four at
//     a time: scores in fp32 (row j's in lane j), their weights, their mix. Rows of other branches are not read;
//   W_UV: head output d = sum_r W[d, r] mix[r] on MFMA, wave w rows 16 w .., its W operands requested at the
//     start (EARLY, one workgroup per CU) or after the merge; the mix enters as three bf16 planes (24 bits), plane
//     p of node j as column TN p + j.
// The output is written as the bf16 hi | lo planes that o_proj's launch takes.
template <int FMT, bool EARLY>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(EARLY ? 2 : 4))) void k_tree_combine(TreeCombArgs a) {
    constexpr int R = 512, DR = 64, NH = 16;
    constexpr int TN = EARLY ? 4 : 8, CB = TN / 4;  // nodes at most, blocks of 16 columns
    const int tn = EARLY ? a.tn : TN;
    __shared__ __attribute__((aligned(16))) uint8_t xs[CB * 16 * 1024];  // column c's words of 8: word ^ (c & 15)
    __shared__ __attribute__((aligned(16))) float red[EARLY ? 8 : 1][R];
    const int tid = threadIdx.x, l = tid & 63, n = l & 15, g = l >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % NH, first = blockIdx.x / NH * tn;
    // this lane's entries of the tables
    const TreeRows q = a.t.s[l];
    const int seq4 = ((const int *)a.nd.seq)[l], parent4 = ((const int *)a.nd.parent)[l];  // four nodes a lane
    const uint16_t *wrow = a.kv_b + ((size_t)h * (a.DN + 128) + a.DN + 16 * w + n) * R + 8 * g;
    v4i wa[16];
    if constexpr (EARLY)
#pragma unroll
        for (int kb = 0; kb < 16; ++kb) wa[kb] = *(const v4i *)(wrow + 32 * kb);
    const int wpn = 8 / tn, j = w / wpn, u = w % wpn;  // node of the workgroup, turn
    const int k = min(first + j, a.n - 1);
    const int b = (tree_lane(seq4, k >> 2) >> (8 * (k & 3))) & 255;
    const TreeRows s{tree_lane(q.a, b), tree_lane(q.b, b), tree_lane(q.c, b), tree_lane(q.ctx, b), tree_lane(q.node0, b),
                     tree_lane(q.part0, b), tree_lane(q.ns, b)};
    const int ns = s.ns, i0 = k - s.node0;
    const float *P = a.part + (size_t)(s.part0 + i0 * ns) * (NH * (R + 2));
    constexpr size_t stride = NH * (R + 2);
    const float *Pm = P + NH * R + h, *Pa = P + h * R + 4 * l;

    // ---- the path's requests (the node's first wave): the head's query, the first four rows
    uint64_t mask = 0;  // bit i: node i of the tree is on the path
    for (int i = i0; i >= 0;) {
        mask |= (uint64_t)1 << i;
        const int z = s.node0 + i;
        i = (int8_t)(tree_lane(parent4, z >> 2) >> (8 * (z & 3)));
    }
    const int np = __builtin_popcountll(mask);
    struct Row {  // four + four latents and a key element of a row, as stored
        v4f f0, f1;
        uint2 h0, h1;
        int q0, q1;
        float sc, key;
    };
    auto ask = [&](size_t row, Row &x) __attribute__((always_inline)) {
        if constexpr (FMT == kFmtQ8) {
            const int8_t *p = (const int8_t *)s.a + row * R + 4 * l;
            x.q0 = *(const int *)p;
            x.q1 = *(const int *)(p + 256);
            x.sc = ((const float *)s.b)[row];
        } else if constexpr (FMT == kFmtF32) {
            const float *p = (const float *)s.a + row * R + 4 * l;
            x.f0 = *(const v4f *)p;
            x.f1 = *(const v4f *)(p + 256);
        } else {
            const uint16_t *p = (const uint16_t *)s.a + row * R + 4 * l;
            x.h0 = *(const uint2 *)p;
            x.h1 = *(const uint2 *)(p + 256);
        }
        x.key = tree_key<FMT>(s, row, DR, l);
    };
    auto lat = [&](const Row &x, v4f &x0, v4f &x1) __attribute__((always_inline)) {
        if constexpr (FMT == kFmtQ8) {
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                x0[z] = (float)(int8_t)(x.q0 >> (8 * z)) * x.sc;
                x1[z] = (float)(int8_t)(x.q1 >> (8 * z)) * x.sc;
            }
        } else if constexpr (FMT == kFmtF32) {
            x0 = x.f0;
            x1 = x.f1;
        } else {
            auto up = [](uint2 h) {
                return v4f{__uint_as_float(h.x << 16), __uint_as_float(h.x & 0xffff0000u), __uint_as_float(h.y << 16),
                           __uint_as_float(h.y & 0xffff0000u)};
            };
            x0 = up(x.h0);
            x1 = up(x.h1);
        }
    };
    // four rows of the path at a time; behind its end its last row again
    int lastrow = 0;
    auto four = [&](uint64_t &m, Row *x) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (m) lastrow = __builtin_ctzll(m);
            m &= m - 1;
            ask((size_t)s.ctx + lastrow, x[r]);
        }
    };
    Row x[4];
    v4f q0, q1;
    float qk = 0.f;
    uint64_t left = mask;
    if (u == 0) {
        const float *qr = a.qf + ((size_t)k * NH + h) * (R + DR);
        q0 = *(const v4f *)(qr + 4 * l);
        q1 = *(const v4f *)(qr + 256 + 4 * l);
        qk = qr[R + l];
        four(left, x);
    }
    // ---- the history's splits, 64 at a time (split s0 + l's maximum and sum in lane l), running maximum
    float mh = -INFINITY, den = 0.f;
    v4f c0 = {0.f, 0.f, 0.f, 0.f}, c1 = c0;
    for (int s0 = 0; s0 < ns; s0 += 64) {
        const int top = min(64, ns - s0);
        const float *pm = Pm + (size_t)(s0 + min(l, top - 1)) * stride;
        const float ms = pm[0], ls = pm[NH];
        auto get = [&](int t, v4f *y0, v4f *y1) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < kTcAhead; ++r) {
                const float *p = Pa + (size_t)(s0 + min(t + r * wpn, top - 1)) * stride;
                y0[r] = *(const v4f *)p;
                y1[r] = *(const v4f *)(p + 256);
            }
        };
        v4f y0[kTcAhead], y1[kTcAhead];
        get(u, y0, y1);
        const float mn = fmaxf(mh, wave_max(ms));
        const float al = __expf(mh - mn), e = l < top ? __expf(ms - mn) : 0.f;
        mh = mn;
        den = fmaf(den, al, ls * e);
        c0 *= al;
        c1 *= al;
        for (int t = u; t < top; t += kTcAhead * wpn) {
            if (t != u) get(t, y0, y1);
#pragma unroll
            for (int r = 0; r < kTcAhead; ++r) {
                if (t + r * wpn >= top) break;
                const float wt = lane_f32(e, t + r * wpn);
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    c0[z] = fmaf(y0[r][z], wt, c0[z]);
                    c1[z] = fmaf(y1[r][z], wt, c1[z]);
                }
            }
        }
    }
    den = wave_sum(den);
    // ---- the path
    float mp = -INFINITY, lp = 0.f;
    v4f p0 = {0.f, 0.f, 0.f, 0.f}, p1 = p0;
    if (u == 0) {
        float sc = -INFINITY;
        for (int t = 0; t < np; t += 4) {
            if (t > 0) four(left, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v4f x0, x1;
                lat(x[r], x0, x1);
                float v = qk * x[r].key;
#pragma unroll
                for (int z = 0; z < 4; ++z) v = fmaf(q1[z], x1[z], fmaf(q0[z], x0[z], v));
                v = wave_sum(v) * a.smscale;
                if (l == t + r && t + r < np) sc = v;
            }
        }
        mp = wave_max(sc);
        const float e = l < np ? __expf(sc - mp) : 0.f;
        lp = wave_sum(e);
        left = mask;
        for (int t = 0; t < np; t += 4) {
            if (np > 4) four(left, x);  // four rows or fewer are still here
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (t + r >= np) break;
                v4f x0, x1;
                lat(x[r], x0, x1);
                const float wt = lane_f32(e, t + r);
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    p0[z] = fmaf(x0[z], wt, p0[z]);
                    p1[z] = fmaf(x1[z], wt, p1[z]);
                }
            }
        }
    }
    if constexpr (!EARLY)
#pragma unroll
        for (int kb = 0; kb < 16; ++kb) wa[kb] = *(const v4i *)(wrow + 32 * kb);
    if (EARLY && wpn > 1) {  // the node's waves in turn order
        *(v4f *)&red[w][4 * l] = c0;
        *(v4f *)&red[w][256 + 4 * l] = c1;
        __syncthreads();
        if (u == 0)
            for (int t = 1; t < wpn; ++t) {
                c0 += *(const v4f *)&red[w + t][4 * l];
                c1 += *(const v4f *)&red[w + t][256 + 4 * l];
            }
    }
    if (u == 0) {
        const float M = fmaxf(mh, mp);
        const float eh = ns > 0 ? __expf(mh - M) : 0.f, ep = __expf(mp - M);
        const float inv = 1.0f / fmaf(den, eh, lp * ep);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const v4f c = half ? c1 : c0, p = half ? p1 : p0;
            v4f x;
#pragma unroll
            for (int z = 0; z < 4; ++z) x[z] = fmaf(c[z], eh, p[z] * ep) * inv;
#pragma unroll
            for (int pl = 0; pl < 3; ++pl) {
                const v2bf b0 = __builtin_convertvector((v2f{x[0], x[1]}), v2bf), b1 = __builtin_convertvector((v2f{x[2], x[3]}), v2bf);
                const int col = TN * pl + j;
                *(int2 *)(xs + col * 1024 + 16 * ((32 * half + (l >> 1)) ^ (col & 15)) + 8 * (l & 1)) =
                    int2{__builtin_bit_cast(int, b0), __builtin_bit_cast(int, b1)};
                x -= v4f{(float)b0.x, (float)b0.y, (float)b1.x, (float)b1.y};
            }
        }
    }
    __syncthreads();
    v4f acc[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) acc[cb] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < 16; ++kb)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
            acc[cb] = mfma_bf16(__builtin_bit_cast(v8bf, wa[kb]), *(const v8bf *)(xs + (16 * cb + n) * 1024 + 16 * ((4 * kb + g) ^ n)), acc[cb]);
    // columns j, TN + j, 2 TN + j are the planes of node j (columns without one are not used)
    const int node = first + n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // TN = 4: row_ror:12, row_ror:8: lanes n + 4, n + 8
        const float mid = TN == 4 ? dpp_f32<0x12C>(acc[0][i]) : dpp_f32<0x128>(acc[0][i]);
        const float low = TN == 4 ? dpp_f32<0x128>(acc[0][i]) : acc[CB - 1][i];
        const float v = acc[0][i] + (mid + low);
        if (n < tn && node < a.n) {
            uint16_t hi, lo;
            split_bf16(v, hi, lo);
            const size_t o = (size_t)node * (NH * 128) + h * 128 + 16 * w + 4 * g + i;
            a.hos[o] = hi;
            a.hos[a.plane + o] = lo;
        }
    }
}

// Y (+)= the partials of the k quarters in their order, a word of four a thread: 2 us at 20 nodes, 5 at 256 (10 MB),
// a launch's latency.
__global__ __launch_bounds__(256) void k_tree_sum(float *Y, const float *P, size_t pstride, size_t n4, int acc) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n4) return;
    v4f p[kGemvKs];
#pragma unroll
    for (int q = 0; q < kGemvKs; ++q) p[q] = *(const v4f *)(P + q * pstride + 4 * i);
    const v4f y = acc ? *(const v4f *)(Y + 4 * i) : v4f{0.f, 0.f, 0.f, 0.f};
    v4f s = p[0];
#pragma unroll
    for (int q = 1; q < kGemvKs; ++q) s += p[q];
    *(v4f *)(Y + 4 * i) = acc ? y + s : s;
}
hipError_t launch_tree_sum(hipStream_t st, float *Y, const float *P, size_t pstride, size_t n, bool accumulate) {
    if (n == 0 || n % 4 || pstride % 4 || (uintptr_t)Y % 16 || (uintptr_t)P % 16) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_tree_sum, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, st, Y, P, pstride, n / 4, accumulate ? 1 : 0);
    return hipGetLastError();
}

// Nodes per workgroup and rows per split.
// nm: 4 share a chunk's staging among twice the queries and overlap it with the products; 2 start sooner,
// waste less of a small tree, and two workgroups a CU cover each other's waits. In chunks' times of the
// former, four take kThStart4 / 10 + X4 / CUs and two kThStart2 / 10 + r X2 / (2 CUs), r = 1.2 (Q8 1.1), X the
// chunks times the workgroups that share them: the lesser is taken. History and combine together, 2 / 4 nodes a
// workgroup (FP32, BF16, Q8): 400 rows x 7 nodes 20 / 24, 18 / 22, 20 / 26 us; 9000 x 13 43 / 45, 35 / 36, 37 / 40;
//   32768 x 8 62 / 59, 44 / 44, 45 / 48; 32768 x 16 99 / 90, 62 / 59, 62 / 61; of several trees, of at most so
//   many nodes each, four of 8192 x 16 75 / 73, 49 / 50, 50 / 53; eight of 4096 x 24 100 / 93, 64 / 61, 64 / 64; two of
//   16384 x 64 259 / 218, 139 / 123, 135 / 125; eight of 32768 x 2 126 / 153, 79 / 87, 61 / 88.
// rows: one chunk a split where that makes at most kThFew workgroups, else a multiple of the chunk, at least
// kThMin. A launch of k rounds of workgroups takes about k (chunks + start), and the combine about one chunk's
// time for each kThJoin splits of a sequence: for each k up to kThRounds the fewest rows that make k rounds
// (or the rows at which fewer splits gain less than they cost), and of these the shortest. kThFew, history and
// combine of 4 nodes per workgroup, one chunk against two (FP32, BF16, Q8): 400 rows x 7 nodes (26 workgroups)
// 23.8 / 26.5, 22.5 / 23.0, 24.1 / 25.3 us; 1400 x 8 (88) 28.3 / 28.3, 26.3 / 25.0, 28.3 / 26.9; 2048 x 8 (128)
// 30.3 / 30.0, 28.8 / 26.3, 30.9 / 28.7.
constexpr int kThFew = 64, kThMin = 64, kThMax = 1 << 19, kThRounds = 4, kThStart4 = 47, kThStart2 = 34, kThJoin = 64;
int plan_tree(int fmt, const Dims &d, TreeTable &t, int ncu) {
    const bool kimi = d.NH == 16 && d.R == 512 && d.DR == 64 && d.DV == 128;
    int longest = 0;
    for (int b = 0; b < t.n; ++b) longest = std::max(longest, t.s[b].ctx);
    auto splits = [](long ctx, long r) { return (ctx + r - 1) / r; };
    auto groups = [&](long chunks, int nm) {
        long n = 0;
        for (int b = 0; b < t.n; ++b) n += (t.s[b].count + nm - 1) / nm * splits(t.s[b].ctx, chunks * kThCh);
        return n;
    };
    const long four = 20 * groups(1, 4) + 2L * ncu * kThStart4, two = (fmt == kFmtQ8 ? 11 : 12) * groups(1, 2) + 2L * ncu * kThStart2;
    t.nm = !kimi ? 0 : four < two ? 4 : 2;
    long best = kThMin / kThCh;  // in chunks
    if (t.nm) {
        const long places = (long)ncu * (t.nm == 2 ? 2 : 1), start = t.nm == 2 ? kThStart2 : kThStart4;
        // at most kThMax rows: offsets within a split stay below 2^31 bytes
        const long all = splits(longest, kThCh), least = groups(1, t.nm) <= kThFew * (4 / t.nm) ? 1 : kThMin / kThCh;
        long cost = LONG_MAX, hi = std::max(least, std::min<long>(all, kThMax / kThCh)), even = least;
        while (even * even * kThJoin < all && even < hi) ++even;
        for (int k = 1; k <= kThRounds; ++k) {
            long lo = least, up = hi;
            while (lo < up) {  // groups() does not increase with the chunks
                const long mid = (lo + up) / 2;
                if (groups(mid, t.nm) <= k * places) up = mid;
                else lo = mid + 1;
            }
            const long r = std::max(lo, even);
            const long c = k * (10 * r + start) + 10 * splits(all, r) / kThJoin;
            if (c < cost) {
                cost = c;
                best = r;
            }
            hi = lo;  // more rounds need no more rows
            if (lo == least) break;
        }
    }
    int part = 0;
    t.units = 0;
    for (int b = 0; b < t.n; ++b) {
        TreeSeq &s = t.s[b];
        s.rps = (int)(best * kThCh);
        s.ns = t.nm ? (int)splits(s.ctx, s.rps) : 0;
        s.tiles = t.nm ? (s.count + t.nm - 1) / t.nm : 1;
        s.part0 = part;
        s.unit0 = t.units;
        part += s.count * (t.nm ? s.ns : 1);
        t.units += s.ns * s.tiles;
    }
    return part;
}

template <int FMT>
static void tree_launch(hipStream_t st, const TreeArgs &a, unsigned grid) {
    if (a.t.nm == 2) hipLaunchKernelGGL((k_tree_hist<FMT, 2>), dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_tree_hist<FMT, 4>), dim3(grid), dim3(512), 0, st, a);
}

static bool tree_table_ok(int fmt, const TreeTable &t, const Dims &d, bool kimi) {
    if (t.n < 1 || t.n > kMaxBatch || t.nodes < 1 || t.nodes > kTreeGroup) return false;
    if (fmt != kFmtQ8 && fmt != kFmtF32 && fmt != kFmtBF16) return false;
    if (!kimi) return t.nm == 0 && d.R <= 256 * kTgCols && d.DR <= 256;
    return (t.nm == 4 || t.nm == 2) && d.NH == 16 && d.R == 512 && d.DR == 64 && d.DV == 128;
}

hipError_t launch_tree_history(hipStream_t st, int fmt, const TreeTable &t, const Dims &d, const DecodeWork &w) {
    if (!tree_table_ok(fmt, t, d, true)) return hipErrorInvalidValue;
    if (t.units == 0) return hipSuccess;  // no history
    const unsigned grid = 8u * (unsigned)((t.units + 7) / 8);
    const TreeArgs a{t, w.qf, w.part, 1.0f / sqrtf((float)d.QD)};
    if (fmt == kFmtQ8) tree_launch<kFmtQ8>(st, a, grid);
    else if (fmt == kFmtF32) tree_launch<kFmtF32>(st, a, grid);
    else tree_launch<kFmtBF16>(st, a, grid);
    return hipGetLastError();
}

hipError_t launch_tree_combine(hipStream_t st, int fmt, const TreeTable &t, const TreeNodes &nd, const Dims &d,
                               const uint16_t *kv_b, const DecodeWork &w) {
    if (!tree_table_ok(fmt, t, d, true)) return hipErrorInvalidValue;
    TreeCombArgs a{tree_rows(t), nd, w.qf, w.part, kv_b, w.hos, (size_t)t.nodes * d.HO, 1.0f / sqrtf((float)d.QD), d.DN, t.nodes, 1};
    // Nodes per workgroup: enough workgroups for the CUs first, then W_UV (128 KB a workgroup) shared by more. 8
    // nodes (W_UV requested after the merge, two workgroups a CU) against 4: 80 nodes 13.7 / 17.0 us, 128 15.6 /
    // 18.1, 168 19.4 / 26.4, 256 22.4 / 33.9 (BF16).
    a.tn = t.nodes <= 16 ? 1 : t.nodes <= 32 ? 2 : t.nodes <= 64 ? 4 : 8;
    const dim3 grid((unsigned)((t.nodes + a.tn - 1) / a.tn * 16));
    const bool early = a.tn < 8;  // one workgroup per CU
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(512), 0, st, a); };
    if (fmt == kFmtQ8) early ? go(k_tree_combine<kFmtQ8, true>) : go(k_tree_combine<kFmtQ8, false>);
    else if (fmt == kFmtF32) early ? go(k_tree_combine<kFmtF32, true>) : go(k_tree_combine<kFmtF32, false>);
    else early ? go(k_tree_combine<kFmtBF16, true>) : go(k_tree_combine<kFmtBF16, false>);
    return hipGetLastError();
}

static_assert(sizeof(TreeCombArgs) <= 4096 && sizeof(TreeNodeArgs) <= 4096 && sizeof(TreeArgs) <= 4096, "kernel arguments");
static_assert(kTreeGroup == 4 * 64, "four nodes a lane");

hipError_t launch_tree_generic(hipStream_t st, int fmt, const TreeTable &t, const TreeNodes &nd, const Dims &d,
                               const DecodeWork &w) {
    if (!tree_table_ok(fmt, t, d, false)) return hipErrorInvalidValue;
    const TreeNodeArgs a{tree_rows(t), nd, w.qf, w.part, 1.0f / sqrtf((float)d.QD), d.NH, d.R, d.DR};
    const dim3 grid((unsigned)(t.nodes * d.NH));
    if (fmt == kFmtQ8) hipLaunchKernelGGL(k_tree_generic<kFmtQ8>, grid, dim3(256), 0, st, a);
    else if (fmt == kFmtF32) hipLaunchKernelGGL(k_tree_generic<kFmtF32>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_tree_generic<kFmtBF16>, grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

// ================================================================ rows =================

// Bytes [lo, hi) from src to n destinations (stride: the next one's pointer), all with the alignment of lo
// to 16 (bases of hipMalloc and equal offsets), hi - lo at most kForkChunk: whole 16-byte words through
// registers, read once, then the ends byte by byte.
// Bytes of an array one block copies: 8 KB is two words a thread, which keeps every CU's loads and stores
// mixed with its neighbours'. Measured, one read for 4 copies of 32768 Q8 rows / 6 copies of rows behind a
// shared prefix, BF16: 4 KB 21.2 / 14.3 us, 8 KB 20.2 / 13.8, 16 KB 20.8 / 15.2, 32 KB 27.6 / 24.2; one read
// for each copy (32 KB): 24.7 / 15.0. Non-temporal words: 25.0 against 20.9 us in the kernel.
constexpr size_t kForkChunk = 8192;
constexpr int kForkWords = kForkChunk / 16 / 256;
__device__ __forceinline__ void copy_range(void *const *dst, int stride, int n, const uint8_t *src, size_t lo, size_t hi) {
    const size_t a = (lo + 15) & ~(size_t)15, b = hi & ~(size_t)15;
    const int tid = threadIdx.x;
    if (a < b) {
        v4i v[kForkWords];
#pragma unroll
        for (int i = 0; i < kForkWords; ++i) {
            const size_t x = a + 16 * (size_t)(256 * i + tid);
            if (x < b) v[i] = *(const v4i *)(src + x);
        }
        for (int d = 0; d < n; ++d) {
            uint8_t *p = (uint8_t *)dst[d * stride];
#pragma unroll
            for (int i = 0; i < kForkWords; ++i) {
                const size_t x = a + 16 * (size_t)(256 * i + tid);
                if (x < b) *(v4i *)(p + x) = v[i];
            }
        }
    }
    const size_t e0 = a < b ? a : hi, e1 = a < b ? b : hi;  // ends: [lo, e0) and [e1, hi)
    for (int d = 0; d < n; ++d) {
        uint8_t *p = (uint8_t *)dst[d * stride];
        for (size_t i = lo + tid; i < e0; i += 256) p[i] = src[i];
        for (size_t i = e1 + tid; i < hi; i += 256) p[i] = src[i];
    }
}

// Block (x, y): chunk x of the arrays of run y (pairs with one source and one range, which a launch takes
// together), cut at multiples of kForkChunk one after another.
__global__ __launch_bounds__(256) void k_fork(ForkTable t) {
    const int first = t.run[blockIdx.y], n = t.run[blockIdx.y + 1] - first;
    const ForkDesc &f = t.d[first];
    size_t c = blockIdx.x;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        if (t.e[k] == 0) continue;
        const size_t lo = (size_t)f.r0 * t.e[k], hi = (size_t)f.r1 * t.e[k], base = lo & ~(kForkChunk - 1);
        const size_t m = (hi - base + kForkChunk - 1) / kForkChunk;
        if (c < m) {
            const size_t x = base + c * kForkChunk;
            copy_range(&f.dst[k], sizeof(ForkDesc) / sizeof(void *), n, (const uint8_t *)f.src[k], x > lo ? x : lo,
                       x + kForkChunk < hi ? x + kForkChunk : hi);
            return;
        }
        c -= m;
    }
}

hipError_t launch_fork(hipStream_t st, ForkTable &t) {
    if (t.n < 1 || t.n > kForkBatch) return hipErrorInvalidValue;
    size_t most = 0;
    int runs = 0;
    for (int i = 0; i < t.n; ++i) {
        const ForkDesc &f = t.d[i];
        if (i > 0 && f.src[0] == t.d[i - 1].src[0] && f.r0 == t.d[i - 1].r0 && f.r1 == t.d[i - 1].r1) continue;
        t.run[runs++] = (uint8_t)i;
        size_t n = 0;
        for (int k = 0; k < 3; ++k) {
            if (t.e[k] == 0) continue;
            const size_t lo = (size_t)f.r0 * t.e[k], hi = (size_t)f.r1 * t.e[k];
            n += (hi - (lo & ~(kForkChunk - 1)) + kForkChunk - 1) / kForkChunk;
        }
        most = std::max(most, n);
    }
    t.run[runs] = (uint8_t)t.n;
    if (most < 1 || most > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_fork, dim3((unsigned)most, (unsigned)runs), dim3(256), 0, st, t);
    return hipGetLastError();
}

// Moves one array's rows, at most 128 columns of `U`-wide words at a time: every row of the path is read
// before the first is written, each thread holding up to kAcceptRows words of one column. (Sources and
// destinations overlap, but only within a column.) Latency bound: 20 states' paths of 17 nodes, Q8, 3.4 us,
// 8.7 with a thread per column and eight rows in flight.
constexpr int kAcceptThreads = 512, kAcceptRows = kTreeNodes / (kAcceptThreads / 128);
template <class U>
__device__ __forceinline__ void move_rows(void *p, int e, const AcceptDesc &d) {
    const int words = e / (int)sizeof(U);
    U *base = (U *)p + (size_t)d.start * words;
    int lg = 0;
    while (lg < 7 && (1 << lg) < words) ++lg;  // columns of a round: a power of two
    const int first = threadIdx.x >> lg, step = kAcceptThreads >> lg;
    for (int c0 = 0; c0 < words; c0 += 1 << lg) {
        const int c = c0 + (threadIdx.x & ((1 << lg) - 1));
        U v[kAcceptRows];
#pragma unroll
        for (int q = 0; q < kAcceptRows; ++q) {
            const int i = first + q * step;
            if (i < d.n && c < words) v[q] = base[(size_t)d.path[i] * words + c];
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < kAcceptRows; ++q) {
            const int i = first + q * step;
            if (i < d.n && c < words) base[(size_t)i * words + c] = v[q];
        }
    }
}

// One block per state and array.
__global__ __launch_bounds__(kAcceptThreads) void k_accept(AcceptTable t) {
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
    hipLaunchKernelGGL(k_accept, dim3((unsigned)t.n, 3), dim3(kAcceptThreads), 0, st, t);
    return hipGetLastError();
}

}  // namespace kvl
