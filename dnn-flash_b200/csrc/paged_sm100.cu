// paged_sm100.cu -- kernels of the paged key-value cache: attention of one new token, appending
// tokens and copying pages (include/odf_paged_sm100.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <math.h>

#include <algorithm>

#include "paged_internal.h"
#include "sm100_ptx.cuh"

namespace odf {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Decode workspace: a counter per CTA, then two partial results per CTA.
constexpr size_t kDecodeCounterBytes = 2048;

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

// ------------------------------------------------------------------------------ decode attention
//
// What bounds it is the cache: every visible key and value is read once (2 d e bytes a key and
// kv-head) against 4 d FLOP per query head, at most a few dozen FLOP a byte, so the kernel is built
// around keeping loads in flight and the arithmetic behind them is one m16n8k16 product per 16
// keys (S = Q K^T, then O += P V, the query heads of one kv-head as the 16 rows).  tcgen05 would
// want 128 rows; there are at most 16, and the warp-level product keeps up (at d = 128 a key costs two
// of them, against 22 clocks that its 512 bytes take at the SM's share of HBM).
//
// Work: an item is (sequence, kv-head, 16 query heads); its visible keys are cut into slices of 16.  The slices
// of all items in a row are dealt to the CTAs in equal consecutive runs, whatever the lengths, by a
// prefix sum over the lengths that every CTA does for itself.  A run holds pieces of one or
// several items; an item that lies in one run is written out directly, the pieces of one that
// does not go to the workspace as fp32 O, max and sum, and the CTA that is last to finish (a
// counter that wraps to zero) joins them in order, so the result does not depend on who that is.
//
// Inside a piece the warps take slices in turn, each with a softmax of its own (running max and sum,
// O in registers) and a ring of its own in shared memory, filled by cp.async kStages - 1 slices
// ahead, across piece borders: no barrier between warps until a piece ends and their parts are joined.
constexpr int kDecodeWarps = 4;
constexpr int kDecodeThreads = kDecodeWarps * 32;
constexpr int kDecodeMaxCtas = 2 * 148;  // two per SM
constexpr int kSlice = 16;               // keys
constexpr int kRowsMax = 16;             // query heads of an item
constexpr int kMinSlices = 16;           // fewest slices worth a CTA of their own
constexpr int kAhead = 2;                // slices whose page ids are asked for before their load
constexpr int kFewItems = 4;             // up to a quarter of the CTAs: a CTA per piece
constexpr int kMergeCols = 32;           // columns of O joined at a time
constexpr int kMergeStride = kMergeCols + 8;  // floats: 8 banks from row to row

template <int D, bool kE4M3>
struct DecodeCfg {
    static constexpr int kRowBytes = D * (kE4M3 ? 1 : 2);
    static constexpr int kTileBytes = kSlice * kRowBytes;   // K or V of a slice
    static constexpr int kStageBytes = 2 * kTileBytes;
    // 24 KB a warp: with two CTAs of four warps, 128 KB of loads in flight on the SM behind the
    // slice that is being computed
    static constexpr int kStages = kStageBytes >= 8192 ? 3 : kStageBytes >= 4096 ? 6 : 8;
    static constexpr int kChunks = kRowBytes / 16;          // 16-byte chunks of a row
    static constexpr int kOffMerge = kDecodeWarps * kStages * kStageBytes;
    static constexpr int kOffStats = kOffMerge + kDecodeWarps * kRowsMax * kMergeStride * 4;
    static constexpr int kOffMask = kOffStats + 2 * kDecodeWarps * kRowsMax * 4;
    static constexpr int kOffPlan = kOffMask + kDecodeWarps * kStages * 4;
    static constexpr int kSmemBytes = kOffPlan + 64 + kDecodeWarps * 8;
    static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs per SM");
};

// Chunk c of row r lies at chunk c ^ swizzle(r): eight consecutive rows then hold one chunk index in
// different banks.
template <int D, bool kE4M3>
__device__ __forceinline__ int swizzle(int r) {
    if constexpr (DecodeCfg<D, kE4M3>::kChunks == 4) return (r >> 1) & 3;
    return r & 7;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
// D[16 x 8] += A[16 x 16] B[16 x 8], fp32 sums, bf16 or f16 operands.
template <bool kHalf>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (kHalf)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four e4m3 values as two pairs of f16 (exact).
__device__ __forceinline__ void e4m3x4_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__host__ __device__ constexpr int64_t run_start(int64_t cta, int64_t total, int64_t ctas) { return cta * total / ctas; }
// The CTA whose run holds slice s.
__device__ __forceinline__ int run_owner(int64_t s, int64_t total, int64_t ctas) {
    return static_cast<int>(((s + 1) * ctas - 1) / total);
}

// Walks a CTA's run piece by piece: slices [s0, s1) of item r of sequence b.
struct RunCursor {
    int b, r, s0, s1;
    int64_t left;  // slices of the run after this piece
    Visible vis;
    int n;         // slices of the item
    __device__ __forceinline__ void enter(const DecodeArgs& a) {
        vis = visible_keys(a, __ldg(a.lens + b));
        n = max(1, (vis.count + kSlice - 1) / kSlice);
    }
    __device__ __forceinline__ void cut() {
        s1 = static_cast<int>(min(static_cast<int64_t>(n), s0 + left));
        left -= s1 - s0;
    }
    __device__ __forceinline__ bool next(const DecodeArgs& a) {
        if (left <= 0) return false;
        s0 = 0;
        if (++r == a.items_per_seq) {
            r = 0;
            ++b;
            enter(a);
        }
        cut();
        return true;
    }
};

template <int D, bool kE4M3>
__global__ void __launch_bounds__(kDecodeThreads, 2) paged_decode_kernel(const __grid_constant__ DecodeArgs a) {
    using Cfg = DecodeCfg<D, kE4M3>;
    constexpr int kStages = Cfg::kStages;
    constexpr int kSteps = D / 16;   // products of S per 8 keys
    constexpr int kBlocks = D / 8;   // column blocks of O
    // 8-bit path: weights as f16 times 2^15, which keeps 11 bits of every weight down to 2^-29 of the
    // row's largest (and something down to 2^-39)
    constexpr float kShift = kE4M3 ? 15.0f : 0.0f;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    float* merge = reinterpret_cast<float*>(smem + Cfg::kOffMerge);
    float* stat_m = reinterpret_cast<float*>(smem + Cfg::kOffStats);
    float* stat_l = stat_m + kDecodeWarps * kRowsMax;
    uint32_t* masks = reinterpret_cast<uint32_t*>(smem + Cfg::kOffMask) + warp * kStages;

    // ---- the run of this CTA
    RunCursor cur;
    int64_t total = 0, first = 0;  // slices of all items; this CTA's first one
    int ctas = 0;
    int few_piece = -1, few_pieces = 0;  // few items: which piece of its item this CTA has, of how many
    {
        int64_t* plan = reinterpret_cast<int64_t*>(smem + Cfg::kOffPlan);
        int64_t* wsum = plan + 4;
        const int per = (a.batch + kDecodeThreads - 1) / kDecodeThreads;
        const int b0 = min(a.batch, static_cast<int>(threadIdx.x) * per), b1 = min(a.batch, b0 + per);
        // Sum of `mine` over all threads, and over those before this one.
        auto scan = [&](int64_t mine, int64_t* before) {
            int64_t incl = mine;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += o;
            }
            if (lane == 31) wsum[warp] = incl;
            __syncthreads();
            int64_t all = 0;
            *before = incl - mine;
#pragma unroll
            for (int w = 0; w < kDecodeWarps; ++w) {
                if (w < warp) *before += wsum[w];
                all += wsum[w];
            }
            __syncthreads();
            return all;
        };
        auto slices_of = [&](int b) {
            const Visible v = visible_keys(a, __ldg(a.lens + b));
            return max(1, (v.count + kSlice - 1) / kSlice);
        };
        int64_t mine = 0, before;
        for (int b = b0; b < b1; ++b) mine += slices_of(b);
        mine *= a.items_per_seq;
        total = scan(mine, &before);
        const int64_t items = static_cast<int64_t>(a.batch) * a.items_per_seq;
        if (items * kFewItems <= gridDim.x) {
            // few items: every piece has a CTA of its own, an item's pieces even
            const int64_t room = gridDim.x - items;
            const int64_t len = max(static_cast<int64_t>(kMinSlices), (total + room - 1) / room);
            mine = 0;
            for (int b = b0; b < b1; ++b) mine += (slices_of(b) + len - 1) / len * a.items_per_seq;
            ctas = static_cast<int>(scan(mine, &before));
            if (static_cast<int>(blockIdx.x) >= ctas) return;
            if (static_cast<int>(blockIdx.x) >= before && static_cast<int>(blockIdx.x) < before + mine) {
                for (int b = b0;; ++b) {
                    const int pieces = static_cast<int>((slices_of(b) + len - 1) / len);
                    const int64_t all = static_cast<int64_t>(pieces) * a.items_per_seq;
                    if (blockIdx.x < before + all) {
                        const int at = static_cast<int>(blockIdx.x - before);
                        plan[0] = b;
                        plan[1] = at / pieces;
                        plan[2] = at % pieces;
                        plan[3] = pieces;
                        break;
                    }
                    before += all;
                }
            }
            __syncthreads();
            cur.b = static_cast<int>(plan[0]);
            cur.r = static_cast<int>(plan[1]);
            few_piece = static_cast<int>(plan[2]);
            few_pieces = static_cast<int>(plan[3]);
            cur.enter(a);
            const int even = (cur.n + few_pieces - 1) / few_pieces;
            cur.s0 = min(cur.n, few_piece * even);
            cur.s1 = min(cur.n, cur.s0 + even);
            cur.left = 0;
        } else {
            const int64_t worth = (total + kMinSlices - 1) / kMinSlices;
            ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), worth));
            if (static_cast<int>(blockIdx.x) >= ctas) return;
            first = run_start(blockIdx.x, total, ctas);
            if (first >= before && first < before + mine) {
                for (int b = b0;; ++b) {
                    const int n = slices_of(b);
                    const int64_t all = static_cast<int64_t>(n) * a.items_per_seq;
                    if (first < before + all) {
                        plan[0] = b;
                        plan[1] = (first - before) / n;
                        plan[2] = (first - before) % n;
                        break;
                    }
                    before += all;
                }
            }
            __syncthreads();
            cur.b = static_cast<int>(plan[0]);
            cur.r = static_cast<int>(plan[1]);
            cur.s0 = static_cast<int>(plan[2]);
            cur.left = run_start(blockIdx.x + 1, total, ctas) - first;
            cur.enter(a);
            cur.cut();
        }
    }

    // ---- loads: this warp's slices s0 + warp, s0 + warp + 4, ... of every piece, in order
    const uint32_t ring = ptx::smem_u32(smem) + warp * (kStages * Cfg::kStageBytes);
    RunCursor ld = cur;
    int ld_s = ld.s0 + warp;
    int ld_slot = 0;  // ring slot of the next load
    // The slices after the next load, whose page ids are on their way: lanes 0-15 stand for the keys' K
    // rows, 16-31 for their V rows.  slot_in_page -1: key not seen; head -1: no slice left.
    int page[kAhead], slot_in_page[kAhead], head[kAhead];
    auto seek = [&](int i) {
        head[i] = -1;
        while (ld_s >= ld.s1) {
            if (!ld.next(a)) return;
            ld_s = ld.s0 + warp;
        }
        head[i] = ld.r / a.row_tiles;
        const int u = ld_s * kSlice + (lane & 15);
        slot_in_page[i] = -1;
        if (u < ld.vis.count) {
            const int j = ld.vis.key(u);
            const int at = static_cast<int>(fast_div(static_cast<uint32_t>(j), a.c.fd_page));
            slot_in_page[i] = j - at * a.c.page_size;
            page[i] = __ldg(a.c.table + ld.b * a.c.table_stride + at);
        }
        ld_s += kDecodeWarps;
    };
    auto load = [&]() {
        if (head[0] >= 0) {
            int64_t off = -1;
            if (slot_in_page[0] >= 0) {
                if (page[0] < 0 || page[0] >= a.c.num_pages)
                    bad_page(a.c);
                else if (lane < 16)
                    off = page[0] * a.c.k_page + head[0] * a.c.k_head + slot_in_page[0] * a.c.k_slot;
                else
                    off = page[0] * a.c.v_page + head[0] * a.c.v_head + slot_in_page[0] * a.c.v_slot;
            }
            const uint32_t seen = __ballot_sync(0xffffffffu, off >= 0);
            if (lane == 0) masks[ld_slot] = seen & 0xffffu;
            constexpr int kRowsPer = 32 / Cfg::kChunks;  // rows per instruction
            const int c = lane % Cfg::kChunks;
            const uint32_t dst = ring + ld_slot * Cfg::kStageBytes;
#pragma unroll
            for (int i = 0; i < kSlice / kRowsPer; ++i) {
                const int row = i * kRowsPer + lane / Cfg::kChunks;
                const uint32_t at = dst + row * Cfg::kRowBytes + ((c ^ swizzle<D, kE4M3>(row)) << 4);
                const int64_t ko = __shfl_sync(0xffffffffu, off, row);
                const int64_t vo = __shfl_sync(0xffffffffu, off, 16 + row);
                // rows that are not seen read as zeros (their bytes are not touched)
                cp_async16(at, a.c.k + (ko < 0 ? 0 : ko + c * 16), ko < 0 ? 0 : 16);
                cp_async16(at + Cfg::kTileBytes, a.c.v + (vo < 0 ? 0 : vo + c * 16), vo < 0 ? 0 : 16);
            }
            ld_slot = ld_slot + 1 == kStages ? 0 : ld_slot + 1;
#pragma unroll
            for (int i = 0; i + 1 < kAhead; ++i) {
                page[i] = page[i + 1];
                slot_in_page[i] = slot_in_page[i + 1];
                head[i] = head[i + 1];
            }
            seek(kAhead - 1);
        }
        cp_async_commit();  // an empty group when there is nothing left, so that the count below holds
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) seek(i);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) load();

    int slot = 0;  // ring slot of the next slice to compute
    int64_t item0 = first - cur.s0;  // slice number, over all items, of the item's first
    for (;;) {
        const int hk = cur.r / a.row_tiles;
        const int row0 = (cur.r - hk * a.row_tiles) * kRowsMax;  // first query head of the item, within the group
        const int rows = min(kRowsMax, a.group - row0);
        const int h0 = hk * a.group + row0;

        // ---- Q as the A operand of S = Q K^T: rows g and g + 8
        uint32_t qf[kSteps][4];
        float unit[2] = {1.0f, 1.0f};  // 8-bit path: what one unit of S is worth, by row
        {
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + cur.b * a.q_b + h0 * a.q_h;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int row = g + 8 * hf;
                const bool ok = row < rows;
                const __nv_bfloat16* qr = q + (ok ? row : 0) * a.q_h;
                if constexpr (!kE4M3) {
#pragma unroll
                    for (int kk = 0; kk < kSteps; ++kk) {
                        qf[kk][hf] = ok ? __ldg(reinterpret_cast<const uint32_t*>(qr + kk * 16 + 2 * t)) : 0u;
                        qf[kk][2 + hf] = ok ? __ldg(reinterpret_cast<const uint32_t*>(qr + kk * 16 + 8 + 2 * t)) : 0u;
                    }
                } else {
                    // lane t holds the D/4 consecutive features whose 8-bit keys it reads; as f16, scaled
                    // by a power of two that puts the row's largest at 2^14 (exact down to 2^-30 of it)
                    uint2 w[kSteps];
                    float mx = 0.0f;
#pragma unroll
                    for (int kk = 0; kk < kSteps; ++kk) {
                        w[kk] = ok ? __ldg(reinterpret_cast<const uint2*>(qr + (D / 4) * t + 4 * kk)) : make_uint2(0u, 0u);
                        mx = fmaxf(mx, fmaxf(fmaxf(fabsf(__uint_as_float(w[kk].x << 16)), fabsf(__uint_as_float(w[kk].x & 0xFFFF0000u))),
                                             fmaxf(fabsf(__uint_as_float(w[kk].y << 16)), fabsf(__uint_as_float(w[kk].y & 0xFFFF0000u)))));
                    }
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    // exponent of the largest, kept where 2^(14 - e) and its inverse are normal
                    int e = static_cast<int>(__float_as_uint(mx) >> 23) - 127;
                    e = mx == 0.0f || e > 127 ? 14 : max(e, -100);
                    const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
                    unit[hf] = __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
#pragma unroll
                    for (int kk = 0; kk < kSteps; ++kk) {
                        qf[kk][hf] = pack_half2(__uint_as_float(w[kk].x << 16) * up, __uint_as_float(w[kk].x & 0xFFFF0000u) * up);
                        qf[kk][2 + hf] = pack_half2(__uint_as_float(w[kk].y << 16) * up, __uint_as_float(w[kk].y & 0xFFFF0000u) * up);
                    }
                }
            }
        }
        float slope[2] = {0.0f, 0.0f};
        if (a.has_alibi) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int h = h0 + g + 8 * hf;
                if (g + 8 * hf < rows)
                    slope[hf] = a.alibi_generated ? exp2f(-8.0f * static_cast<float>(h + 1) / static_cast<float>(a.heads_q))
                                                  : a.alibi_slopes[h];
            }
        }
        const float ks = a.c.k_scale ? __ldg(a.c.k_scale + hk) : 1.0f;
        const bool capped = a.softcap > 0.0f;
        // score = S * mul + slope * (j - p): log2 units, or units of the soft-cap
        const float into = capped ? a.inv_softcap : kLog2e;
        float mul[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            mul[hf] = a.scale * unit[hf] * ks * into;
            slope[hf] *= into;
        }

        float o[kBlocks][4];
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

        for (int s = cur.s0 + warp; s < cur.s1; s += kDecodeWarps) {
            cp_async_wait<kStages - 2>();
            __syncwarp();
            load();  // into the slot whose slice every lane has finished
            const uint32_t kt = ring + slot * Cfg::kStageBytes;
            const uint32_t vt = kt + Cfg::kTileBytes;
            const uint32_t seen = masks[slot];
            slot = slot + 1 == kStages ? 0 : slot + 1;

            // S[16 rows x 16 keys]: keys 2t, 2t + 1 of the lower and the upper eight
            float sc[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
            if constexpr (!kE4M3) {
                const int key = ((lane >> 4) << 3) + (lane & 7);
                const uint32_t at = kt + key * Cfg::kRowBytes + ((((lane >> 3) & 1) ^ swizzle<D, kE4M3>(key)) << 4);
#pragma unroll
                for (int kk = 0; kk < kSteps; ++kk) {
                    uint32_t b[4];
                    ldmatrix4(at ^ (kk << 5), b);
                    mma16816<false>(sc[0], qf[kk], b[0], b[1]);
                    mma16816<false>(sc[1], qf[kk], b[2], b[3]);
                }
            } else {
#pragma unroll
                for (int nb = 0; nb < 2; ++nb) {
                    const int key = nb * 8 + g;
#pragma unroll
                    for (int c = 0; c < kSteps / 4; ++c) {
                        const int chunk = (kSteps / 4) * t + c;
                        const uint4 w = lds128(kt + key * Cfg::kRowBytes + ((chunk ^ swizzle<D, kE4M3>(key)) << 4));
                        uint32_t b0, b1;
                        e4m3x4_to_half(w.x, b0, b1);
                        mma16816<true>(sc[nb], qf[4 * c + 0], b0, b1);
                        e4m3x4_to_half(w.y, b0, b1);
                        mma16816<true>(sc[nb], qf[4 * c + 1], b0, b1);
                        e4m3x4_to_half(w.z, b0, b1);
                        mma16816<true>(sc[nb], qf[4 * c + 2], b0, b1);
                        e4m3x4_to_half(w.w, b0, b1);
                        mma16816<true>(sc[nb], qf[4 * c + 3], b0, b1);
                    }
                }
            }

            // score mods, mask, running max
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = nb * 8 + 2 * t + (i & 1);
                    float x = sc[nb][i] * mul[i >> 1];
                    if (a.has_alibi)
                        x += slope[i >> 1] * static_cast<float>(cur.vis.key(s * kSlice + key) - (cur.vis.len - 1));
                    if (capped) x = a.softcap * kLog2e * tanhf(x);
                    x = (seen >> key) & 1u ? x : -INFINITY;
                    sc[nb][i] = x;
                    mx[i >> 1] = fmaxf(mx[i >> 1], x);
                }
            }
            bool moved = false;
            float alpha[2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 1));
                mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 2));
                const float mn = fmaxf(m[hf], mx[hf]);
                alpha[hf] = mn > m[hf] ? ptx::ex2(m[hf] - mn) : 1.0f;
                moved |= mn > m[hf];
                m[hf] = mn;
            }
            if (__any_sync(0xffffffffu, moved)) {
                l[0] *= alpha[0];
                l[1] *= alpha[1];
#pragma unroll
                for (int j = 0; j < kBlocks; ++j) {
                    o[j][0] *= alpha[0];
                    o[j][1] *= alpha[0];
                    o[j][2] *= alpha[1];
                    o[j][3] *= alpha[1];
                }
            }
            const float ref[2] = {(m[0] == -INFINITY ? 0.0f : m[0]) - kShift, (m[1] == -INFINITY ? 0.0f : m[1]) - kShift};
            // P in the operand's type; l sums it before that rounding
            uint32_t p[4];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = ptx::ex2(sc[nb][i] - ref[i >> 1]);
                l[0] += e[0] + e[1];
                l[1] += e[2] + e[3];
                p[2 * nb] = kE4M3 ? pack_half2(e[0], e[1]) : ptx::pack_bf16x2(e[0], e[1]);
                p[2 * nb + 1] = kE4M3 ? pack_half2(e[2], e[3]) : ptx::pack_bf16x2(e[2], e[3]);
            }

            // O += P V
            if constexpr (!kE4M3) {
                const int key = (((lane >> 3) & 1) << 3) + (lane & 7);
                const uint32_t at = vt + key * Cfg::kRowBytes + (((lane >> 4) ^ swizzle<D, kE4M3>(key)) << 4);
#pragma unroll
                for (int dd = 0; dd < kSteps; ++dd) {
                    uint32_t b[4];
                    ldmatrix4_trans(at ^ (dd << 5), b);
                    mma16816<false>(o[2 * dd], p, b[0], b[1]);
                    mma16816<false>(o[2 * dd + 1], p, b[2], b[3]);
                }
            } else {
                // column n of block j is feature (D/8) n + j: lane g reads D/8 consecutive features of
                // keys 2t, 2t+1, 2t+8, 2t+9 and pairs the keys' bytes feature by feature
                uint32_t w[4][D / 32];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = 2 * t + (i & 1) + 8 * (i >> 1);
                    if constexpr (D == 128) {
                        const uint4 x = lds128(vt + key * Cfg::kRowBytes + ((g ^ swizzle<D, kE4M3>(key)) << 4));
                        w[i][0] = x.x;
                        w[i][1] = x.y;
                        w[i][2] = x.z;
                        w[i][3] = x.w;
                    } else {
                        const uint2 x = lds64(vt + key * Cfg::kRowBytes + (((g >> 1) ^ swizzle<D, kE4M3>(key)) << 4) + (g & 1) * 8);
                        w[i][0] = x.x;
                        w[i][1] = x.y;
                    }
                }
#pragma unroll
                for (int q4 = 0; q4 < D / 32; ++q4) {
                    uint32_t b0[4], b1[4];
                    e4m3x4_to_half(__byte_perm(w[0][q4], w[1][q4], 0x5140), b0[0], b0[1]);
                    e4m3x4_to_half(__byte_perm(w[0][q4], w[1][q4], 0x7362), b0[2], b0[3]);
                    e4m3x4_to_half(__byte_perm(w[2][q4], w[3][q4], 0x5140), b1[0], b1[1]);
                    e4m3x4_to_half(__byte_perm(w[2][q4], w[3][q4], 0x7362), b1[2], b1[3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) mma16816<true>(o[4 * q4 + i], p, b0[i], b1[i]);
                }
            }
        }

        // ---- the warps' parts of the piece: a common max, then O in strips of kMergeCols columns
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
            if (t == 0) {
                stat_m[warp * kRowsMax + g + 8 * hf] = m[hf];
                stat_l[warp * kRowsMax + g + 8 * hf] = l[hf];
            }
        }
        __syncthreads();
        const int row = threadIdx.x >> 3;  // of the joined result: 16 rows x 8 threads of 4 columns
        const bool row_ok = row < rows;
        float M = -INFINITY, L = 0.0f, wt[kDecodeWarps];
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) M = fmaxf(M, stat_m[w * kRowsMax + row]);
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) {
            const float mw = stat_m[w * kRowsMax + row];
            wt[w] = mw == -INFINITY ? 0.0f : ptx::ex2(mw - M);
            L += wt[w] * stat_l[w * kRowsMax + row];
        }
        const bool whole = cur.s0 == 0 && cur.s1 == cur.n;
        // partial results: slot 2c + 1 for the item that starts in this run, 2c for one that started before
        float* slots = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + kDecodeCounterBytes);
        constexpr int kSlotFloats = kRowsMax * D + 2 * kRowsMax;
        float* part = slots + (2 * static_cast<int64_t>(blockIdx.x) + (cur.s0 == 0 ? 1 : 0)) * kSlotFloats;
        const float vs = a.c.v_scale ? __ldg(a.c.v_scale + hk) : 1.0f;
        auto write_out = [&](int r, int col, float4 x, float sum) {
            const float inv = sum == 0.0f ? 0.0f : vs / sum;  // a row that sees no key: 0
            x = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
            const int64_t at = cur.b * a.o_b + (h0 + r) * a.o_h + col;
            if (a.o_bf16)
                *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.o) + at) =
                    make_uint2(ptx::pack_bf16x2(x.x, x.y), ptx::pack_bf16x2(x.z, x.w));
            else
                *reinterpret_cast<float4*>(static_cast<float*>(a.o) + at) = x;
        };
        auto write_lse = [&](int r, float mr, float sum) {
            if (a.lse)
                a.lse[static_cast<int64_t>(cur.b) * a.heads_q + h0 + r] =
                    sum == 0.0f ? -INFINITY : (mr + (log2f(sum) - kShift)) * kLn2;
        };
        // A strip is four column blocks: bf16 columns 8 j + n, in order; 8-bit features (D/8) n + j, four
        // in a row for each n.  With at most 8 rows the other half of the buffer takes every second strip.
        const int other = rows <= 8 ? 8 * kMergeStride : 0;
#pragma unroll
        for (int q4 = 0; q4 < kBlocks / 4; ++q4) {
            float* buf = merge + ((q4 & 1) ? other : 0);
            if (q4 > 0 && other == 0) __syncthreads();  // the strip before has been read
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int r = g + 8 * hf;
                float* dst = buf + (warp * kRowsMax + r) * kMergeStride;
                if (r < rows) {
                    if constexpr (kE4M3) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            *reinterpret_cast<float4*>(dst + (2 * t + i) * 4) =
                                make_float4(o[4 * q4][2 * hf + i], o[4 * q4 + 1][2 * hf + i], o[4 * q4 + 2][2 * hf + i],
                                            o[4 * q4 + 3][2 * hf + i]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            *reinterpret_cast<float2*>(dst + 8 * j + 2 * t) = make_float2(o[4 * q4 + j][2 * hf], o[4 * q4 + j][2 * hf + 1]);
                    }
                }
            }
            __syncthreads();
            if (row_ok) {
                const int c4 = threadIdx.x & 7;
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kDecodeWarps; ++w) {
                    const float4 y = *reinterpret_cast<const float4*>(buf + (w * kRowsMax + row) * kMergeStride + 4 * c4);
                    x.x += wt[w] * y.x;
                    x.y += wt[w] * y.y;
                    x.z += wt[w] * y.z;
                    x.w += wt[w] * y.w;
                }
                const int d = kE4M3 ? (D / 8) * c4 + 4 * q4 : kMergeCols * q4 + 4 * c4;
                if (whole)
                    write_out(row, d, x, L);
                else
                    *reinterpret_cast<float4*>(part + row * D + d) = x;
            }
        }
        if (row_ok && (threadIdx.x & 7) == 0) {
            if (whole) {
                write_lse(row, M, L);
            } else {
                part[kRowsMax * D + row] = M;
                part[kRowsMax * D + kRowsMax + row] = L;
            }
        }
        if (!whole) {
            const int c_first = few_piece >= 0 ? static_cast<int>(blockIdx.x) - few_piece : run_owner(item0, total, ctas);
            const int pieces = few_piece >= 0 ? few_pieces : run_owner(item0 + cur.n - 1, total, ctas) - c_first + 1;
            __syncthreads();  // the CTA's part is written, as seen from its first thread
            int* last = reinterpret_cast<int*>(smem + Cfg::kOffPlan);
            if (threadIdx.x == 0) {
                __threadfence();
                const unsigned int old =
                    atomicInc(static_cast<unsigned int*>(a.workspace) + c_first, static_cast<unsigned int>(pieces - 1));
                __threadfence();
                *last = old == static_cast<unsigned int>(pieces - 1);
            }
            __syncthreads();
            const bool join = *last != 0;
            __syncthreads();
            if (join) {
                auto piece = [&](int k) {
                    return slots + (2 * static_cast<int64_t>(c_first + k) + (k == 0 ? 1 : 0)) * kSlotFloats;
                };
                // the pieces' weights by row (8 threads to a row), then O, float4 units of the rows spread
                // over the threads (with few rows, the pieces too) so that many loads are in flight
                constexpr int kHeld = kDecodeWarps * kMergeStride;
                float* wts = merge;  // [min(pieces, kHeld)][kRowsMax]
                float mj = -INFINITY, lj = 0.0f;
#pragma unroll 4
                for (int k = threadIdx.x & 7; k < pieces; k += 8) {
                    const float mk = __ldcg(piece(k) + kRowsMax * D + row);
                    const float lk = __ldcg(piece(k) + kRowsMax * D + kRowsMax + row);
                    if (k < kHeld) wts[k * kRowsMax + row] = mk;
                    const float mn = fmaxf(mj, mk);
                    if (mn != -INFINITY) lj = lj * ptx::ex2(mj - mn) + lk * ptx::ex2(mk - mn);
                    else lj += lk;  // 0, or NaN
                    mj = mn;
                }
#pragma unroll
                for (int off = 4; off > 0; off >>= 1) {
                    const float mo = __shfl_xor_sync(0xffffffffu, mj, off), lo = __shfl_xor_sync(0xffffffffu, lj, off);
                    const float mn = fmaxf(mj, mo);
                    lj = mn == -INFINITY ? lj + lo : lj * ptx::ex2(mj - mn) + lo * ptx::ex2(mo - mn);
                    mj = mn;
                }
                for (int k = threadIdx.x & 7; k < min(pieces, kHeld); k += 8) {
                    const float mk = wts[k * kRowsMax + row];
                    wts[k * kRowsMax + row] = mk == -INFINITY ? 0.0f : ptx::ex2(mk - mj);
                }
                if ((threadIdx.x & 7) == 0) {
                    stat_m[row] = mj;
                    stat_l[row] = lj;
                }
                if (row_ok && (threadIdx.x & 7) == 0) write_lse(row, mj, lj);
                __syncthreads();
                constexpr int kUnitsMax = kRowsMax * (D / 4) / kDecodeThreads;  // per thread
                const int units = rows * (D / 4);
                const int groups = units >= kDecodeThreads ? 1 : kDecodeThreads / units;
                const int grp = static_cast<int>(threadIdx.x) / units;
                const int u0 = groups > 1 ? static_cast<int>(threadIdx.x) - grp * units : static_cast<int>(threadIdx.x);
                float4 x[kUnitsMax];
#pragma unroll
                for (int i = 0; i < kUnitsMax; ++i) x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (grp < groups || groups == 1) {
#pragma unroll 8
                    for (int k = groups > 1 ? grp : 0; k < pieces; k += groups) {
                        const float4* pk = reinterpret_cast<const float4*>(piece(k));
#pragma unroll
                        for (int i = 0; i < kUnitsMax; ++i) {
                            const int u = u0 + i * kDecodeThreads;
                            if (u < units) {
                                const float4 y = __ldcg(pk + u);
                                const int r = u / (D / 4);
                                float w;
                                if (k < kHeld) {
                                    w = wts[k * kRowsMax + r];
                                } else {  // one item over most of the GPU
                                    const float mk = __ldcg(piece(k) + kRowsMax * D + r);
                                    w = mk == -INFINITY ? 0.0f : ptx::ex2(mk - stat_m[r]);
                                }
                                x[i].x += w * y.x;
                                x[i].y += w * y.y;
                                x[i].z += w * y.z;
                                x[i].w += w * y.w;
                            }
                        }
                    }
                }
                if (groups > 1) {
                    __syncthreads();  // the weights have been read
                    float4* sums = reinterpret_cast<float4*>(merge);
                    if (grp < groups) sums[grp * units + u0] = x[0];
                    __syncthreads();
                    if (grp == 0) {
                        for (int k = 1; k < groups; ++k) {
                            const float4 y = sums[k * units + u0];
                            x[0].x += y.x;
                            x[0].y += y.y;
                            x[0].z += y.z;
                            x[0].w += y.w;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < kUnitsMax; ++i) {
                    const int u = u0 + i * kDecodeThreads;
                    if (u < units && (groups == 1 || grp == 0))
                        write_out(u / (D / 4), (u % (D / 4)) * 4, x[i], stat_l[u / (D / 4)]);
                }
                __syncthreads();
            }
        }
        item0 += cur.n;
        if (!cur.next(a)) break;
    }
    cp_async_wait<0>();
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

size_t decode_workspace_bytes(int32_t head_dim) {
    return kDecodeCounterBytes + 2 * sizeof(float) * kDecodeMaxCtas * (static_cast<size_t>(kRowsMax) * head_dim + 2 * kRowsMax);
}

namespace {

template <int D, bool kE4M3>
cudaError_t launch_decode(const DecodeArgs& a, unsigned grid, cudaStream_t stream) {
    constexpr int smem = DecodeCfg<D, kE4M3>::kSmemBytes;
    const cudaError_t e =
        cudaFuncSetAttribute(paged_decode_kernel<D, kE4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    paged_decode_kernel<D, kE4M3><<<grid, kDecodeThreads, smem, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

int launch_paged_decode(DecodeArgs& a, int32_t head_dim, int32_t kv_dtype, cudaStream_t stream, const char** err) {
    static_assert(kDecodeCounterBytes >= kDecodeMaxCtas * sizeof(unsigned int), "a counter per CTA");
    a.row_tiles = (a.group + kRowsMax - 1) / kRowsMax;
    a.items_per_seq = a.c.heads_kv * a.row_tiles;
    // no more CTAs than the page table's room could give work to
    const int64_t room = static_cast<int64_t>(a.c.max_pages) * a.c.page_size;
    int64_t keys = room;
    if (a.window > 0 && static_cast<int64_t>(a.window) + a.sinks < room) keys = static_cast<int64_t>(a.window) + a.sinks;
    const int64_t slices = (keys + kSlice - 1) / kSlice * a.items_per_seq * a.batch;
    // and as many as give every piece of few items one of its own
    const int64_t worth =
        std::max((slices + kMinSlices - 1) / kMinSlices, static_cast<int64_t>(kFewItems) * a.items_per_seq * a.batch);
    const int64_t most = std::min<int64_t>(kDecodeMaxCtas, 2 * static_cast<int64_t>(a.sm_count));
    const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, std::min(most, worth)));
    cudaError_t e;
    if (kv_dtype == ODF_DTYPE_E4M3)
        e = head_dim == 64 ? launch_decode<64, true>(a, grid, stream) : launch_decode<128, true>(a, grid, stream);
    else
        e = head_dim == 64 ? launch_decode<64, false>(a, grid, stream) : launch_decode<128, false>(a, grid, stream);
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
