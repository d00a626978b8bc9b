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

hipError_t launch_tree_attention(hipStream_t st, int fmt, const TreeTable &t, const Dims &d, const DecodeWork &w) {
    if (d.R > 256 * kTgCols || d.DR > 256 || t.n < 1 || t.nodes < 1 || t.nodes > kTreeNodes) return hipErrorInvalidValue;
    TreeArgs a;
    a.t = t;
    a.d = d;
    a.qf = w.qf;
    a.part = w.part;
    a.smscale = 1.0f / sqrtf((float)d.QD);
    const dim3 grid((unsigned)(t.nodes * d.NH));
    if (fmt == kFmtQ8) hipLaunchKernelGGL(k_tree_generic<kFmtQ8>, grid, dim3(256), 0, st, a);
    else if (fmt == kFmtF32) hipLaunchKernelGGL(k_tree_generic<kFmtF32>, grid, dim3(256), 0, st, a);
    else if (fmt == kFmtBF16) hipLaunchKernelGGL(k_tree_generic<kFmtBF16>, grid, dim3(256), 0, st, a);
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
