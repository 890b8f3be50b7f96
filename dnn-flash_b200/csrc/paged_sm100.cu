// paged_sm100.cu -- kernels of the paged key-value cache: attention of one new token, appending
// tokens and copying pages (include/odf_paged_sm100.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <math.h>

#include "paged_internal.h"
#include "sm100_ptx.cuh"

namespace odf {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void bad_page(const PagedView& c) {
    if (c.status) atomicCAS(c.status, 0, ODF_ERR_BAD_PAGE);
}

// The keys that a token at position len - 1 sees, as consecutive indices u in [0, count): the
// first `sinks` of them are keys 0 .. sinks - 1, the others start at `lo`.  A length beyond what
// the page table holds is cut (and reported).
struct Visible {
    int count, sinks, lo, len;
    __device__ __forceinline__ int key(int u) const { return u < sinks ? u : lo + (u - sinks); }
};

__device__ __forceinline__ Visible visible_keys(const DecodeArgs& a, int len) {
    Visible r;
    const int room = a.c.max_pages * a.c.page_size;
    r.len = len < 0 ? 0 : len;
    if (r.len > room) {
        bad_page(a.c);
        r.len = room;
    }
    r.lo = a.window > 0 ? max(0, r.len - a.window) : 0;
    r.sinks = min(a.window > 0 ? a.sinks : 0, r.lo);
    r.count = r.sinks + (r.len - r.lo);
    return r;
}

// Byte offsets of a token's K and V rows of head hk, or -1 with a page id out of range.
__device__ __forceinline__ bool row_offsets(const PagedView& c, const int32_t* table, int j, int hk, int64_t* k, int64_t* v) {
    const int at = static_cast<int>(fast_div(static_cast<uint32_t>(j), c.fd_page));
    const int slot = j - at * c.page_size;
    const int page = __ldg(table + at);
    if (page < 0 || page >= c.num_pages) {
        bad_page(c);
        return false;
    }
    *k = page * c.k_page + hk * c.k_head + slot * c.k_slot;
    *v = page * c.v_page + hk * c.v_head + slot * c.v_slot;
    return true;
}

template <int V>
__device__ __forceinline__ void load_row(const uint8_t* p, int lane, bool e4m3, float* x) {
    if (e4m3) {
        const __nv_fp8_e4m3* s = reinterpret_cast<const __nv_fp8_e4m3*>(p) + lane * V;
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = static_cast<float>(s[i]);
    } else {
        const __nv_bfloat16* s = reinterpret_cast<const __nv_bfloat16*>(p) + lane * V;
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = __bfloat162float(s[i]);
    }
}

// One block per (batch, q-head), a key per warp at a time.
constexpr int kDecodeWarps = 4;

template <int D>
__global__ void __launch_bounds__(kDecodeWarps * 32) paged_decode_kernel(const __grid_constant__ DecodeArgs a, bool e4m3) {
    constexpr int V = D / 32;
    const int b = blockIdx.x / a.heads_q;
    const int h = blockIdx.x - b * a.heads_q;
    const int hk = h / a.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Visible vis = visible_keys(a, __ldg(a.lens + b));
    const int32_t* table = a.c.table + b * a.c.table_stride;
    const float ks = a.c.k_scale ? a.c.k_scale[hk] : 1.0f;
    const float vs = a.c.v_scale ? a.c.v_scale[hk] : 1.0f;
    float slope = 0.0f;
    if (a.has_alibi)
        slope = a.alibi_generated ? exp2f(-8.0f * static_cast<float>(h + 1) / static_cast<float>(a.heads_q)) : a.alibi_slopes[h];
    float q[V], acc[V];
    load_row<V>(reinterpret_cast<const uint8_t*>(static_cast<const __nv_bfloat16*>(a.q) + b * a.q_b + h * a.q_h), lane, false, q);
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (int u = warp; u < vis.count; u += kDecodeWarps) {
        const int j = vis.key(u);
        int64_t ko, vo;
        if (!row_offsets(a.c, table, j, hk, &ko, &vo)) continue;
        float k[V], v[V];
        load_row<V>(a.c.k + ko, lane, e4m3, k);
        load_row<V>(a.c.v + vo, lane, e4m3, v);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        s = s * (a.scale * ks) + slope * static_cast<float>(j - (vis.len - 1));
        if (a.softcap > 0.0f) s = a.softcap * tanhf(s * a.inv_softcap);
        const float mn = fmaxf(m, s);
        const float alpha = m == -INFINITY ? 0.0f : expf(m - mn);
        const float p = expf(s - mn);
        l = l * alpha + p;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = acc[i] * alpha + p * v[i];
        m = mn;
    }
    __shared__ float sm[kDecodeWarps], sl[kDecodeWarps], so[kDecodeWarps][D];
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) so[warp][lane * V + i] = acc[i];
    __syncthreads();
    float mx = -INFINITY, sum = 0.0f;
    for (int w = 0; w < kDecodeWarps; ++w) mx = fmaxf(mx, sm[w]);
    float wt[kDecodeWarps];
    for (int w = 0; w < kDecodeWarps; ++w) {
        wt[w] = sl[w] == 0.0f ? 0.0f : expf(sm[w] - mx);
        sum += wt[w] * sl[w];
    }
    if (threadIdx.x < D) {
        float o = 0.0f;
        for (int w = 0; w < kDecodeWarps; ++w)
            if (sl[w] != 0.0f) o += wt[w] * so[w][threadIdx.x];
        o = vis.count > 0 ? o / sum * vs : 0.0f;
        const int64_t at = b * a.o_b + h * a.o_h + threadIdx.x;
        if (a.o_bf16)
            static_cast<__nv_bfloat16*>(a.o)[at] = __float2bfloat16_rn(o);
        else
            static_cast<float*>(a.o)[at] = o;
    }
    if (threadIdx.x == 0 && a.lse) a.lse[static_cast<int64_t>(b) * a.heads_q + h] = vis.count > 0 ? mx + logf(sum) : -INFINITY;
}

// A thread per 16 bytes of new row: K, then V.
__device__ __forceinline__ uint32_t quantise4(const float* x, float scale) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r |= static_cast<uint32_t>(__nv_cvt_float_to_fp8(__fdiv_rn(x[i], scale), __NV_SATFINITE, __NV_E4M3)) << (8 * i);
    return r;
}

template <int D>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ AppendArgs a, bool e4m3) {
    constexpr int kVecs = D / 8;
    const int64_t total = static_cast<int64_t>(a.batch) * a.tokens * a.c.heads_kv * kVecs;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int c = static_cast<int>(i % kVecs);
        int64_t r = i / kVecs;
        const int t = static_cast<int>(r % a.tokens);
        r /= a.tokens;
        const int hk = static_cast<int>(r % a.c.heads_kv);
        const int b = static_cast<int>(r / a.c.heads_kv);
        if (a.counts && t >= __ldg(a.counts + b)) continue;
        const int64_t pos = static_cast<int64_t>(__ldg(a.starts + b)) + t;
        if (pos < 0 || pos >= static_cast<int64_t>(a.c.max_pages) * a.c.page_size) {
            bad_page(a.c);
            continue;
        }
        int64_t ko, vo;
        if (!row_offsets(a.c, a.c.table + b * a.c.table_stride, static_cast<int>(pos), hk, &ko, &vo)) continue;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(which ? a.v : a.k) +
                                       (which ? b * a.v_b + hk * a.v_h + t * a.v_t : b * a.k_b + hk * a.k_h + t * a.k_t) + c * 8;
            uint8_t* dst = which ? a.c.v + vo : a.c.k + ko;
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(src));
            if (!e4m3) {
                reinterpret_cast<uint4*>(dst)[c] = w;
            } else {
                const float* sp = which ? a.c.v_scale : a.c.k_scale;
                const float scale = sp ? __ldg(sp + hk) : 1.0f;
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
                float x[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[2 * e] = __uint_as_float(u[e] << 16);
                    x[2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u);
                }
                reinterpret_cast<uint2*>(dst)[c] = make_uint2(quantise4(x, scale), quantise4(x + 4, scale));
            }
        }
    }
}

// Pairs travel in the launch's parameters.
template <int N>
struct PairList {
    int32_t id[2 * N];
};

template <int N>
__global__ void __launch_bounds__(256) page_copy_kernel(const __grid_constant__ CopyArgs a, const __grid_constant__ PairList<N> list) {
    const int which = blockIdx.z & 1;
    const int layer = blockIdx.z >> 1;
    const int pair = blockIdx.x;
    const int64_t src = list.id[2 * pair] * a.page[which] + layer * a.layer[which];
    const int64_t dst = list.id[2 * pair + 1] * a.page[which] + layer * a.layer[which];
    const int64_t vecs = a.run_bytes[which] / 16;
    const int64_t total = vecs * a.inner[which] * a.outer[which];
    for (int64_t i = static_cast<int64_t>(blockIdx.y) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.y) * blockDim.x) {
        const int64_t run = i / vecs;
        const int64_t o = run / a.inner[which];
        const int64_t off = o * a.outer_stride[which] + (run - o * a.inner[which]) * a.inner_stride[which] + (i - run * vecs) * 16;
        *reinterpret_cast<uint4*>(a.base[which] + dst + off) = *reinterpret_cast<const uint4*>(a.base[which] + src + off);
    }
}

template <int N>
cudaError_t launch_copy(const CopyArgs& a, int64_t first, int64_t count, cudaStream_t stream) {
    PairList<N> list;
    for (int64_t i = 0; i < 2 * count; ++i) list.id[i] = a.pairs[2 * first + i];
    for (int l = 0; l < a.layers; l += 32767) {
        CopyArgs x = a;
        x.pairs = nullptr;
        x.layers = a.layers - l < 32767 ? a.layers - l : 32767;
        for (int w = 0; w < 2; ++w) x.base[w] += l * x.layer[w];
        const dim3 grid(static_cast<unsigned>(count), 4, 2 * x.layers);
        page_copy_kernel<N><<<grid, 256, 0, stream>>>(x, list);
    }
    return cudaGetLastError();
}

}  // namespace

size_t decode_workspace_bytes(int32_t) { return 256; }

int launch_paged_decode(DecodeArgs& a, int32_t head_dim, int32_t kv_dtype, cudaStream_t stream, const char** err) {
    const unsigned grid = static_cast<unsigned>(a.batch) * static_cast<unsigned>(a.heads_q);
    const bool e4m3 = kv_dtype == ODF_DTYPE_E4M3;
    if (head_dim == 64)
        paged_decode_kernel<64><<<grid, kDecodeWarps * 32, 0, stream>>>(a, e4m3);
    else
        paged_decode_kernel<128><<<grid, kDecodeWarps * 32, 0, stream>>>(a, e4m3);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) *err = cudaGetErrorString(e);
    return e == cudaSuccess ? ODF_OK : ODF_ERR_CUDA;
}

int launch_paged_append(AppendArgs& a, int32_t head_dim, int32_t kv_dtype, cudaStream_t stream, const char** err) {
    const bool e4m3 = kv_dtype == ODF_DTYPE_E4M3;
    const int64_t total = static_cast<int64_t>(a.batch) * a.tokens * a.c.heads_kv * (head_dim / 8);
    const int64_t blocks = (total + 255) / 256;
    const unsigned grid = static_cast<unsigned>(blocks < 148 * 16 ? blocks : 148 * 16);
    if (head_dim == 64)
        paged_append_kernel<64><<<grid, 256, 0, stream>>>(a, e4m3);
    else
        paged_append_kernel<128><<<grid, 256, 0, stream>>>(a, e4m3);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) *err = cudaGetErrorString(e);
    return e == cudaSuccess ? ODF_OK : ODF_ERR_CUDA;
}

int launch_page_copy(const CopyArgs& a, cudaStream_t stream, const char** err) {
    cudaError_t e = cudaSuccess;
    for (int64_t first = 0; first < a.n_pairs && e == cudaSuccess;) {
        const int64_t left = a.n_pairs - first;
        const int64_t count = left < 400 ? left : 400;
        e = count <= 16 ? launch_copy<16>(a, first, count, stream) : launch_copy<400>(a, first, count, stream);
        first += count;
    }
    if (e != cudaSuccess) *err = cudaGetErrorString(e);
    return e == cudaSuccess ? ODF_OK : ODF_ERR_CUDA;
}

}  // namespace odf
