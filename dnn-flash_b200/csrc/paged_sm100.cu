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

// Decode workspace: three counters per CTA (one per level of a join), then two partial results per CTA.
constexpr size_t kDecodeCounterBytes = 6144;

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

// ------------------------------------------------------------------------------ decode attention
//
// What bounds it is the cache: every visible key and value is read once (2 d e bytes a key and
// kv-head) against 4 d FLOP per query head, at most a few dozen FLOP a byte, so the kernel is built
// around keeping loads in flight and short chains of arithmetic behind them.
//
// Products are warp-level m16n8k16 with the keys as the 16 rows: S^T = K Q^T, then O^T += V^T P^T, the
// query heads of one kv-head as the 8 columns (one block of them up to 8 heads, else two).  tcgen05 would
// want 128 rows of keys by 8 columns through tensor memory; the warp-level product leaves the tensor
// pipe 9% busy (16% with an 8-bit cache) and needs no hand-over between warps.
//
// 64 sequences of up to 8192 keys, 64/8 heads, three draws of their lengths: 1079, 1132 and 1131 MB of visible keys
// in 165, 172 and 176 us (6.4 to 6.6 TB/s); one sequence of 129 keys 4.5 us in a replayed graph.
//
// Work: an item is (sequence, kv-head, block of query heads); its visible keys are cut into slices of 16 or
// 32.  The slices of all items in a row are dealt to the CTAs in equal consecutive runs, whatever
// the lengths, by a prefix sum over the lengths that every warp does for itself; when items are
// few, or their lengths near enough, each has CTAs of its own.  A run holds pieces of one or several
// items; an item that lies in one run is written out directly, the pieces of one that does not go
// to the workspace as fp32 O, max and sum, and are joined by whichever CTA is last to finish of each group of
// eight (counters that wrap to zero), in an order that does not depend on who that is.
//
// Inside a piece the warps take slices in turn, each with a softmax of its own (running max and sum,
// O in registers) and a ring of its own in shared memory, filled by cp.async kStages - 1 slices
// ahead, across piece borders: no barrier between warps until a piece ends and their parts are joined.
constexpr int kDecodeWarps = 4;
constexpr int kDecodeThreads = kDecodeWarps * 32;
constexpr int kCtasPerSm = 3;            // of one block of query heads; two of two blocks
constexpr int kDecodeMaxCtas = kCtasPerSm * 148;
constexpr int kRowsMax = 16;             // query heads of an item, at most
constexpr int kMinSlices = 8;            // fewest slices worth a CTA of their own (8 sequences of 1024 keys: 13.9 us
                                         // with 16, 12.5 with 8; 1 of 1500: 11.3 and 12.2)
constexpr int kAhead = 2;                // slices whose page ids are asked for before their load (3: level, 3-9% slower
                                         // with an 8-bit cache)
constexpr int kItemCost = 12;            // slices that stream in the time an item takes besides (Q, joining, output);
                                         // of 5, 8, 12 and 20 the best over ragged, short, e4m3 and 16-head batches
constexpr int kFewItems = 4;             // up to a quarter of the CTAs: a CTA per piece
constexpr int kMergeCols = 32;           // columns of O in a strip of the merge buffer
constexpr int kMergeStride = kMergeCols + 4;  // floats: two rows are 8 banks apart
constexpr int kMergeSlots = 16;          // strips of a warp

template <int D, bool kE4M3, int R>
struct DecodeCfg {
    static constexpr int kRows = 8 * R;                     // query heads of an item
    static constexpr int kRowBytes = D * (kE4M3 ? 1 : 2);
    // Keys of a slice: 16 of 256 bytes; 32 shorter ones, which leaves the chain of products, maxima and
    // exponentials of a slice twice the bytes to hide behind
    static constexpr int kSlice = kRowBytes >= 256 ? 16 : 32;
    static constexpr int kTileBytes = kSlice * kRowBytes;   // K or V of a slice
    static constexpr int kStageBytes = 2 * kTileBytes;
    // 16 KB a warp with three CTAs of four warps on an SM, 24 KB with two: 96 or 128 KB of loads in flight on an SM
    // (144 or 160 with 8-bit rows of 64) behind the slices that are being computed.  Three do as well or better wherever their registers
    // allow it (64 ragged sequences of 8-bit rows of 64: 57 us against 66).
    static constexpr int kCtas = R == 1 ? kCtasPerSm : 2;
    static constexpr int kStages = (kCtas == 3 ? 16384 : 24576) / kStageBytes;
    static constexpr int kChunks = kRowBytes / 16;          // 16-byte chunks of a row
    static constexpr int kOffMerge = kDecodeWarps * kStages * kStageBytes;
    static constexpr int kOffStats = kOffMerge + kDecodeWarps * kMergeSlots * kMergeStride * 4;
    static constexpr int kOffMask = kOffStats + 2 * kDecodeWarps * kRowsMax * 4;
    static constexpr int kOffLast = kOffMask + kDecodeWarps * kStages * 4;
    static constexpr int kSmemBytes = kOffLast + 16;
    static constexpr int kSlotFloats = kRows * D + 2 * kRows;  // a partial result
    static_assert(kCtas * (kSmemBytes + 1024) <= 228 * 1024, "CTAs per SM");
};

// Chunk c of row r lies at chunk c ^ swizzle(r): eight consecutive rows then hold one chunk index in
// different banks.
template <int kChunks>
__device__ __forceinline__ int swizzle(int r) {
    if constexpr (kChunks == 4) return (r >> 1) & 3;
    return r & 7;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
// An 8x8 matrix of 16-bit values across the warp, transposed.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Runs of equal length: the first `more` CTAs' are one longer than the others' `len`.
struct Runs {
    int len, more;
    __device__ __forceinline__ int start(int cta) const { return cta * len + min(cta, more); }
    // the CTA whose run holds s
    __device__ __forceinline__ int owner(int s) const {
        const int edge = more * (len + 1);
        return s < edge ? static_cast<int>(static_cast<uint32_t>(s) / static_cast<uint32_t>(len + 1))
                        : more + static_cast<int>(static_cast<uint32_t>(s - edge) / static_cast<uint32_t>(len));
    }
};

// Walks a CTA's run piece by piece: slices [s0, s1) of item r of sequence b.  Runs are measured in slices plus
// kItemCost per item, spent before its first slice.
template <int kSlice>
struct RunCursor {
    int b, r, s0, s1;
    int left;      // of the run after this piece
    bool whole;    // the run is of whole items
    Visible vis;
    int n;         // slices of the item: one at least, so that an empty one is written too
    __device__ __forceinline__ void enter(const DecodeArgs& a) {
        vis = visible_keys(a, __ldg(a.lens + b));
        n = max(1, (vis.count + kSlice - 1) / kSlice);
    }
    // the piece from offset x of the item on; false if the run ends before a slice of it
    __device__ __forceinline__ bool cut(int x) {
        const int end = whole ? n + kItemCost : min(n + kItemCost, x + left);
        left -= end - x;
        s0 = max(0, x - kItemCost);
        s1 = max(0, end - kItemCost);
        return s1 > s0;
    }
    __device__ __forceinline__ bool next(const DecodeArgs& a) {
        if (left <= 0) return false;
        if (++r == a.items_per_seq) {
            r = 0;
            if (++b >= a.batch) return false;  // only with lengths that change under the kernel
            enter(a);
        }
        return cut(0);
    }
};

template <int D, bool kE4M3, int R>
__global__ void __launch_bounds__(kDecodeThreads, DecodeCfg<D, kE4M3, R>::kCtas)
    paged_decode_kernel(const __grid_constant__ DecodeArgs a) {
    using Cfg = DecodeCfg<D, kE4M3, R>;
    constexpr int kRows = Cfg::kRows;
    constexpr int kStages = Cfg::kStages;
    constexpr int kSlice = Cfg::kSlice;
    constexpr int kChunks = Cfg::kChunks;
    constexpr int kKb = kSlice / 16;  // blocks of 16 keys
    constexpr int kSteps = D / 16;    // products of S per block; blocks of 16 columns of O
    // The reference max moves only when a score passes it by more than 2^kLazy, so that most slices need
    // one vote instead of a row maximum.  8-bit path: weights are f16 times 2^7, at most 2^15; all of
    // their 11 bits are kept down to 2^-21 of the reference and something down to 2^-31.
    constexpr float kLazy = 8.0f;
    constexpr float kShift = kE4M3 ? 7.0f : 0.0f;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    float* merge = reinterpret_cast<float*>(smem + Cfg::kOffMerge);
    float* stat_m = reinterpret_cast<float*>(smem + Cfg::kOffStats);
    float* stat_l = stat_m + kDecodeWarps * kRowsMax;
    uint32_t* masks = reinterpret_cast<uint32_t*>(smem + Cfg::kOffMask) + warp * kStages;

    // ---- the run of this CTA; every warp works it out for itself, a lane per batch / 32 sequences
    RunCursor<kSlice> cur;
    Runs runs{0, 0};
    int first = 0;                   // where this CTA's run starts
    int item0 = 0;                   // and its item
    int few_piece = -1, pieces = 0;  // a CTA per piece: which piece of its item this one has, of how many
    {
        const int cta = static_cast<int>(blockIdx.x), grid = static_cast<int>(gridDim.x);
        const int per = (a.batch + 31) / 32;
        const int b0 = min(a.batch, lane * per), b1 = min(a.batch, b0 + per);
        auto slices_of = [&](int b) {
            const Visible v = visible_keys(a, __ldg(a.lens + b));
            return max(1, (v.count + kSlice - 1) / kSlice);
        };
        // sum over the lanes before this one; `all` of every lane
        auto scan = [&](int mine, int& all) {
            int incl = mine;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += o;
            }
            all = __shfl_sync(0xffffffffu, incl, 31);
            return incl - mine;
        };
        int mine = 0, most = 0, total, before = 0;
        if (a.batch == 1) {
            most = slices_of(0);
            total = most * a.items_per_seq;
            mine = lane == 0 ? total : 0;
        } else {
#pragma unroll 4
            for (int b = b0; b < b1; ++b) {
                const int n = slices_of(b);
                mine += n;
                most = max(most, n);
            }
            most = __reduce_max_sync(0xffffffffu, most);
            mine *= a.items_per_seq;
            before = scan(mine, total);
        }
        const int items = a.batch * a.items_per_seq;
        // No item is cut when the longest streams in about the time that cutting items and joining the pieces
        // takes: runs are of whole items; with a CTA for each, items may also be near an even share (with 40
        // for 24, 8 sequences of 1024 keys, 64 slices an item, take 17.4 us, cut 12.5).  The share: a CTA on its
        // own takes some 200 to 300 times as long for a slice as all SMs together.  Measured, both sides, on
        // 606 batches of 112 to 440 items of up to 852 slices, of one length or spread by up to 95% (bf16 and
        // e4m3, d 64 and 128): the rule costs 0.5% over the better side on average (18% at most), with total / 160
        // 3.2% (42%), always cut 8.3% (65%), never 12% (153%).
        const bool uncut = most <= 40;
        const bool whole_items = items <= grid && most <= total / 280 + 24;
        const bool few = whole_items || items <= grid / kFewItems;
        int at_b = 0, at_r = 0, at_s = 0;
        if (whole_items) {
            if (cta >= items) return;
            at_b = static_cast<int>(fast_div(static_cast<uint32_t>(cta), a.fd_items));
            at_r = cta - at_b * a.items_per_seq;
            pieces = 1;
        } else {
            int len = 1;  // few items: slices of a piece, at most
            if (few) {
                len = max(kMinSlices, total / (grid - items) + 1);  // an item's pieces are even
                if (a.batch == 1) {
                    total = (most + len - 1) / len * a.items_per_seq;
                    mine = lane == 0 ? total : 0;
                } else {
                    mine = 0;
                    for (int b = b0; b < b1; ++b) mine += (slices_of(b) + len - 1) / len * a.items_per_seq;
                    before = scan(mine, total);
                }
                if (cta >= total) return;
                first = cta;
            } else {
                total += kItemCost * items;
                mine += kItemCost * (b1 - b0) * a.items_per_seq;
                before += kItemCost * b0 * a.items_per_seq;
                const int ctas = min(grid, (total + kMinSlices + kItemCost - 1) / (kMinSlices + kItemCost));
                if (cta >= ctas) return;
                runs.len = total / ctas;
                runs.more = total - runs.len * ctas;
                first = runs.start(cta);
            }
            // the lane whose sequences hold `first` finds the item and the place (or piece) in it
            const bool here = first >= before && first < before + mine;
            if (here) {
                for (at_b = b0; at_b < b1 - 1; ++at_b) {
                    const int n = few ? (slices_of(at_b) + len - 1) / len : slices_of(at_b) + kItemCost;
                    if (first < before + n * a.items_per_seq) break;
                    before += n * a.items_per_seq;
                }
                const int n = few ? (slices_of(at_b) + len - 1) / len : slices_of(at_b) + kItemCost;
                at_r = min(a.items_per_seq - 1, static_cast<int>(static_cast<uint32_t>(first - before) / static_cast<uint32_t>(n)));
                at_s = first - before - at_r * n;
            }
            const int who = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
            at_b = __shfl_sync(0xffffffffu, at_b, who);
            at_r = __shfl_sync(0xffffffffu, at_r, who);
            at_s = __shfl_sync(0xffffffffu, at_s, who);
            pieces = len;
        }
        cur.b = at_b;
        cur.r = at_r;
        cur.s0 = at_s;
        cur.enter(a);
        cur.whole = false;
        if (few) {
            few_piece = at_s;
            cur.s1 = cur.n;
            cur.left = 0;
            if (!whole_items) {
                pieces = (cur.n + pieces - 1) / pieces;
                const int even = (cur.n + pieces - 1) / pieces;
                cur.s0 = min(cur.n, few_piece * even);
                cur.s1 = min(cur.n, cur.s0 + even);
            }
        } else {
            cur.left = runs.start(cta + 1) - first;
            cur.whole = uncut;
            item0 = first - at_s;
            if (uncut && at_s > 0) {  // the items that start in the run
                cur.left -= cur.n + kItemCost - at_s;
                if (!cur.next(a)) return;
            } else if (!cur.cut(at_s)) {
                return;
            }
        }
    }

    // ---- loads: this warp's slices s0 + warp, s0 + warp + 4, ... of every piece, in order
    const uint32_t ring = ptx::smem_u32(smem) + warp * (kStages * Cfg::kStageBytes);
    RunCursor<kSlice> ld = cur;
    int ld_s = ld.s0 + warp;
    int ld_slot = 0;  // ring slot of the next load
    // The slices after the next load, whose page ids are on their way; a lane stands for the key
    // lane % kSlice.  slot_in_page -1: key not seen; head -1: no slice left.
    int page[kAhead], slot_in_page[kAhead], head[kAhead];
    auto seek = [&](int i) {
        head[i] = -1;
        while (ld_s >= ld.s1) {
            if (!ld.next(a)) return;
            ld_s = ld.s0 + warp;
        }
        head[i] = ld.r / a.row_tiles;
        const int u = ld_s * kSlice + lane % kSlice;
        slot_in_page[i] = -1;
        if (u < ld.vis.count) {
            const int j = ld.vis.key(u);
            const int at = static_cast<int>(fast_div(static_cast<uint32_t>(j), a.c.fd_page));
            slot_in_page[i] = j - at * a.c.page_size;
            page[i] = __ldg(a.c.table + ld.b * a.c.table_stride + at);
        }
        ld_s += kDecodeWarps;
    };
    constexpr uint32_t kNoRow = 0xffffffffu;
    const int chunk = lane % kChunks;
    auto load = [&]() {
        if (head[0] >= 0) {
            // rows in 16-byte units (the host refuses caches past 64 GB)
            uint32_t k_off = kNoRow, v_off = kNoRow;
            if (slot_in_page[0] >= 0) {
                if (page[0] < 0 || page[0] >= a.c.num_pages) {
                    bad_page(a.c);
                } else {
                    k_off = static_cast<uint32_t>(page[0]) * a.k16_page + static_cast<uint32_t>(head[0]) * a.k16_head +
                            static_cast<uint32_t>(slot_in_page[0]) * a.k16_slot;
                    v_off = static_cast<uint32_t>(page[0]) * a.v16_page + static_cast<uint32_t>(head[0]) * a.v16_head +
                            static_cast<uint32_t>(slot_in_page[0]) * a.v16_slot;
                }
            }
            const uint32_t seen = __ballot_sync(0xffffffffu, k_off != kNoRow);
            if (lane == 0) masks[ld_slot] = seen;
            constexpr int kRowsPer = 32 / kChunks;  // rows per instruction
            const uint32_t dst = ring + ld_slot * Cfg::kStageBytes;
#pragma unroll
            for (int i = 0; i < kSlice / kRowsPer; ++i) {
                const int row = i * kRowsPer + lane / kChunks;
                const uint32_t at = dst + row * Cfg::kRowBytes + ((chunk ^ swizzle<kChunks>(row)) << 4);
                const uint32_t ko = __shfl_sync(0xffffffffu, k_off, row);
                const uint32_t vo = __shfl_sync(0xffffffffu, v_off, row);
                // rows that are not seen read as zeros (their bytes are not touched)
                const int bytes = ko == kNoRow ? 0 : 16;
                cp_async16(at, a.c.k + (static_cast<uint64_t>(bytes ? ko + chunk : 0) << 4), bytes);
                cp_async16(at + Cfg::kTileBytes, a.c.v + (static_cast<uint64_t>(bytes ? vo + chunk : 0) << 4), bytes);
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
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) load();

    int slot = 0;  // ring slot of the next slice to compute
    for (;;) {
        const int hk = cur.r / a.row_tiles;
        const int row0 = (cur.r - hk * a.row_tiles) * kRows;  // first query head of the item, within the group
        const int rows = min(kRows, a.group - row0);
        const int h0 = hk * a.group + row0;

        // ---- Q as the B operand of S^T = K Q^T: query head g of each block
        uint32_t qf[R][kSteps][2];
        float unit[R];  // 8-bit path: what one unit of S is worth, for query head g of the block
        {
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + cur.b * a.q_b + h0 * a.q_h;
#pragma unroll
            for (int rb = 0; rb < R; ++rb) {
                const int row = g + 8 * rb;
                const bool ok = row < rows;
                const __nv_bfloat16* qr = q + (ok ? row : 0) * a.q_h;
                unit[rb] = 1.0f;
                if constexpr (!kE4M3) {
#pragma unroll
                    for (int kk = 0; kk < kSteps; ++kk) {
                        qf[rb][kk][0] = ok ? __ldg(reinterpret_cast<const uint32_t*>(qr + kk * 16 + 2 * t)) : 0u;
                        qf[rb][kk][1] = ok ? __ldg(reinterpret_cast<const uint32_t*>(qr + kk * 16 + 8 + 2 * t)) : 0u;
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
                    unit[rb] = __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
#pragma unroll
                    for (int kk = 0; kk < kSteps; ++kk) {
                        qf[rb][kk][0] = pack_half2(__uint_as_float(w[kk].x << 16) * up, __uint_as_float(w[kk].x & 0xFFFF0000u) * up);
                        qf[rb][kk][1] = pack_half2(__uint_as_float(w[kk].y << 16) * up, __uint_as_float(w[kk].y & 0xFFFF0000u) * up);
                    }
                }
            }
        }
        const float ks = a.c.k_scale ? __ldg(a.c.k_scale + hk) : 1.0f;
        const bool capped = a.softcap > 0.0f;
        // score = S * mul + slope * (j - p), in log2 units or in units of the soft-cap; a thread has
        // query heads 2t, 2t + 1 of each block
        const float into = capped ? a.inv_softcap : kLog2e;
        float mul[2 * R], slope[2 * R];
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) {
            const int row = 2 * t + (i & 1) + 8 * (i >> 1);
            const float u = kE4M3 ? __shfl_sync(0xffffffffu, unit[i >> 1], 4 * (2 * t + (i & 1))) : 1.0f;
            mul[i] = a.scale * u * ks * into;
            slope[i] = 0.0f;
            if (a.has_alibi && row < rows) {
                const int h = h0 + row;
                slope[i] = into * (a.alibi_generated ? exp2f(-8.0f * static_cast<float>(h + 1) / static_cast<float>(a.heads_q))
                                                     : a.alibi_slopes[h]);
            }
        }

        // O^T: block j of 16 columns by query heads 2t, 2t + 1 of block rb
        float o[R][kSteps][4];
#pragma unroll
        for (int rb = 0; rb < R; ++rb)
#pragma unroll
            for (int j = 0; j < kSteps; ++j) o[rb][j][0] = o[rb][j][1] = o[rb][j][2] = o[rb][j][3] = 0.0f;
        float m[2 * R], l[2 * R];
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
        }

        for (int s = cur.s0 + warp; s < cur.s1; s += kDecodeWarps) {
            cp_async_wait<kStages - 2>();
            __syncwarp();
            load();  // into the slot whose slice every lane has finished
            const uint32_t kt = ring + slot * Cfg::kStageBytes;
            const uint32_t vt = kt + Cfg::kTileBytes;
            const uint32_t seen = masks[slot];
            slot = slot + 1 == kStages ? 0 : slot + 1;

            // S^T: keys g, g + 8 of each block of 16 by query heads 2t, 2t + 1; the steps of a block sum
            // in kChains chains, so that four or more are under way
            constexpr int kChains = kKb * R >= 4 ? 1 : 4 / (kKb * R);
            float sc[kKb][R][4], chain[kChains][kKb][R][4];
#pragma unroll
            for (int c = 0; c < kChains; ++c)
#pragma unroll
                for (int kb = 0; kb < kKb; ++kb)
#pragma unroll
                    for (int rb = 0; rb < R; ++rb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) chain[c][kb][rb][i] = 0.0f;
#pragma unroll
            for (int kb = 0; kb < kKb; ++kb) {
                if constexpr (!kE4M3) {
                    const int key = kb * 16 + (lane & 15);
                    const uint32_t at = kt + key * Cfg::kRowBytes + (((lane >> 4) ^ swizzle<kChunks>(key)) << 4);
#pragma unroll
                    for (int kk = 0; kk < kSteps; ++kk) {
                        uint32_t k[4];
                        ldmatrix4(at ^ (kk << 5), k);
#pragma unroll
                        for (int rb = 0; rb < R; ++rb)
                            mma16816<false>(chain[kk % kChains][kb][rb], k, qf[rb][kk][0], qf[rb][kk][1]);
                    }
                } else {
                    const int key = kb * 16 + g;
#pragma unroll
                    for (int c = 0; c < kSteps / 4; ++c) {
                        const int ch = (kSteps / 4) * t + c;
                        const uint4 w0 = lds128(kt + key * Cfg::kRowBytes + ((ch ^ swizzle<kChunks>(key)) << 4));
                        const uint4 w1 = lds128(kt + (key + 8) * Cfg::kRowBytes + ((ch ^ swizzle<kChunks>(key + 8)) << 4));
                        const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t k[4];
                            e4m3x4_to_half(x0[i], k[0], k[2]);
                            e4m3x4_to_half(x1[i], k[1], k[3]);
#pragma unroll
                            for (int rb = 0; rb < R; ++rb)
                                mma16816<true>(chain[i % kChains][kb][rb], k, qf[rb][4 * c + i][0], qf[rb][4 * c + i][1]);
                        }
                    }
                }
            }

            // score mods, mask, and whether a score passes the reference max
            float mx[2 * R];
#pragma unroll
            for (int i = 0; i < 2 * R; ++i) mx[i] = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < kKb; ++kb) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = kb * 16 + g + 8 * (i >> 1);
                    const bool on = (seen >> key) & 1u;
#pragma unroll
                    for (int rb = 0; rb < R; ++rb) {
                        const int h = 2 * rb + (i & 1);
                        float x = chain[0][kb][rb][i];
#pragma unroll
                        for (int c = 1; c < kChains; ++c) x += chain[c][kb][rb][i];
                        x *= mul[h];
                        if (a.has_alibi) x += slope[h] * static_cast<float>(cur.vis.key(s * kSlice + key) - (cur.vis.len - 1));
                        if (capped) x = a.softcap * kLog2e * tanhf(x);
                        x = on ? x : -INFINITY;
                        sc[kb][rb][i] = x;
                        mx[h] = fmaxf(mx[h], x);
                    }
                }
            }
            bool passes = false;
#pragma unroll
            for (int i = 0; i < 2 * R; ++i) passes |= mx[i] > m[i] + kLazy;
            if (__any_sync(0xffffffffu, passes)) {
#pragma unroll
                for (int i = 0; i < 2 * R; ++i) {
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], off));
                    float alpha = 1.0f;
                    if (mx[i] > m[i]) {
                        alpha = ptx::ex2(m[i] - mx[i]);
                        m[i] = mx[i];
                    }
                    l[i] *= alpha;
#pragma unroll
                    for (int j = 0; j < kSteps; ++j) {
                        o[i >> 1][j][i & 1] *= alpha;
                        o[i >> 1][j][2 + (i & 1)] *= alpha;
                    }
                }
            }
            float ref[2 * R];
#pragma unroll
            for (int i = 0; i < 2 * R; ++i) ref[i] = (m[i] == -INFINITY ? 0.0f : m[i]) - kShift;
            // P in the operand's type, transposed to keys 2t, 2t + 1 by query head g; l sums it before that
            // rounding
            uint32_t p[kKb][R][2];
#pragma unroll
            for (int kb = 0; kb < kKb; ++kb) {
#pragma unroll
                for (int rb = 0; rb < R; ++rb) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const float e0 = ptx::ex2(sc[kb][rb][2 * hf] - ref[2 * rb]);
                        const float e1 = ptx::ex2(sc[kb][rb][2 * hf + 1] - ref[2 * rb + 1]);
                        l[2 * rb] += e0;
                        l[2 * rb + 1] += e1;
                        p[kb][rb][hf] = movmatrix_trans(kE4M3 ? pack_half2(e0, e1) : ptx::pack_bf16x2(e0, e1));
                    }
                }
            }

            // O^T += V^T P^T
#pragma unroll
            for (int kb = 0; kb < kKb; ++kb) {
                if constexpr (!kE4M3) {
                    const int key = kb * 16 + ((lane >> 4) << 3) + (lane & 7);
                    const uint32_t at = vt + key * Cfg::kRowBytes + ((((lane >> 3) & 1) ^ swizzle<kChunks>(key)) << 4);
#pragma unroll
                    for (int j = 0; j < kSteps; ++j) {
                        uint32_t v[4];
                        ldmatrix4_trans(at ^ (j << 5), v);
#pragma unroll
                        for (int rb = 0; rb < R; ++rb) mma16816<false>(o[rb][j], v, p[kb][rb][0], p[kb][rb][1]);
                    }
                } else {
                    // rows g and g + 8 of block j are columns (D/8) g + 2j and + 1: lane g reads D/8 consecutive
                    // ones of keys 2t, 2t+1, 2t+8, 2t+9 and pairs the keys' bytes column by column
                    uint32_t w[4][D / 32];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = kb * 16 + 2 * t + (i & 1) + 8 * (i >> 1);
                        if constexpr (D == 128) {
                            const uint4 x = lds128(vt + key * Cfg::kRowBytes + ((g ^ swizzle<kChunks>(key)) << 4));
                            w[i][0] = x.x;
                            w[i][1] = x.y;
                            w[i][2] = x.z;
                            w[i][3] = x.w;
                        } else {
                            const uint2 x =
                                lds64(vt + key * Cfg::kRowBytes + (((g >> 1) ^ swizzle<kChunks>(key)) << 4) + (g & 1) * 8);
                            w[i][0] = x.x;
                            w[i][1] = x.y;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < kSteps; ++j) {
                        uint32_t v[4];
                        const uint32_t sel = j & 1 ? 0x7362 : 0x5140;
                        e4m3x4_to_half(__byte_perm(w[0][j >> 1], w[1][j >> 1], sel), v[0], v[1]);
                        e4m3x4_to_half(__byte_perm(w[2][j >> 1], w[3][j >> 1], sel), v[2], v[3]);
#pragma unroll
                        for (int rb = 0; rb < R; ++rb) mma16816<true>(o[rb][j], v, p[kb][rb][0], p[kb][rb][1]);
                    }
                }
            }
        }

        // ---- the warps' parts of the piece: a common max, then O in strips of kMergeCols columns
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], off);
            if (g == 0) {
                const int row = 2 * t + (i & 1) + 8 * (i >> 1);
                stat_m[warp * kRowsMax + row] = m[i];
                stat_l[warp * kRowsMax + row] = l[i];
            }
        }
        __syncthreads();
        // a thread's place in the joined strips: 16 slots x 8 threads of 4 columns; a slot is a query head, with
        // one block of them in one of two strips
        const int strip_of = R == 1 ? threadIdx.x >> 6 : 0;
        const int row = (threadIdx.x >> 3) & (kRows - 1);
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
        constexpr int kSlotFloats = Cfg::kSlotFloats;
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
        // A strip is two blocks of 16 columns: in order in a bf16 cache; columns (D/8) g + 4 strip .. + 3 for
        // each g in an 8-bit one.
        constexpr int kPass = 2 / R;  // strips at a time
#pragma unroll
        for (int q0 = 0; q0 < D / kMergeCols; q0 += kPass) {
            if (q0 > 0) __syncthreads();  // the strips before have been read
#pragma unroll
            for (int qq = 0; qq < kPass; ++qq) {
#pragma unroll
                for (int i = 0; i < 2 * R; ++i) {
                    const int r = 2 * t + (i & 1) + 8 * (i >> 1);
                    const int j = 2 * (q0 + qq);
                    float* dst = merge + (warp * kMergeSlots + 8 * qq + r) * kMergeStride;
                    const float x0 = o[i >> 1][j][i & 1], x1 = o[i >> 1][j][2 + (i & 1)];
                    const float x2 = o[i >> 1][j + 1][i & 1], x3 = o[i >> 1][j + 1][2 + (i & 1)];
                    if constexpr (kE4M3) {
                        *reinterpret_cast<float4*>(dst + 4 * g) = make_float4(x0, x1, x2, x3);
                    } else {
                        dst[g] = x0;
                        dst[g + 8] = x1;
                        dst[g + 16] = x2;
                        dst[g + 24] = x3;
                    }
                }
            }
            __syncthreads();
            if (row_ok) {
                const int c4 = threadIdx.x & 7;
                const int strip = q0 + strip_of;
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kDecodeWarps; ++w) {
                    const float4 y = *reinterpret_cast<const float4*>(
                        merge + (w * kMergeSlots + (threadIdx.x >> 3)) * kMergeStride + 4 * c4);
                    x.x += wt[w] * y.x;
                    x.y += wt[w] * y.y;
                    x.z += wt[w] * y.z;
                    x.w += wt[w] * y.w;
                }
                const int d = kE4M3 ? (D / 8) * c4 + 4 * strip : kMergeCols * strip + 4 * c4;
                if (whole)
                    write_out(row, d, x, L);
                else
                    *reinterpret_cast<float4*>(part + row * D + d) = x;
            }
        }
        if (row_ok && strip_of == 0 && (threadIdx.x & 7) == 0) {
            if (whole) {
                write_lse(row, M, L);
            } else {
                part[kRows * D + row] = M;
                part[kRows * D + kRows + row] = L;
            }
        }
        if (!whole) {
            int index = few_piece;  // of this piece
            if (few_piece < 0) {
                const int c_first = runs.owner(item0 + kItemCost);
                index = static_cast<int>(blockIdx.x) - c_first;
                pieces = runs.owner(item0 + kItemCost + cur.n - 1) - c_first + 1;
            }
            // Joined in a tree of eights: whoever is last to finish of a group of eight pieces joins them into the slot of
            // the group's first, then stands for the group among the next eight.  Each step waits twice (about
            // 0.8 us) for other SMs' results: the counter, and all of the group's loads at once.
            const int c_first = static_cast<int>(blockIdx.x) - index;
            float* p0 = slots + 2 * static_cast<int64_t>(c_first) * kSlotFloats;  // piece k > 0: 2 k slots on
            unsigned int* counter = static_cast<unsigned int*>(a.workspace) + c_first;
            int* last = reinterpret_cast<int*>(smem + Cfg::kOffLast);
            int stride = 1;
#pragma unroll 1
            for (;;) {
                const int base = index & ~7;           // the group's first piece, of `pieces` that are `stride` apart
                const int n = min(8, pieces - base);
                float* group = p0 + (base == 0 ? kSlotFloats : 2 * base * stride * kSlotFloats);
                auto piece = [&](int k) { return k == 0 ? group : p0 + 2 * (base + k) * stride * kSlotFloats; };
                if (n > 1) {
                    __syncthreads();  // the CTA's part is written, as seen from its first thread
                    if (threadIdx.x == 0) {
                        __threadfence();
                        const unsigned int old = atomicInc(counter + base * stride, static_cast<unsigned int>(n - 1));
                        __threadfence();
                        *last = old == static_cast<unsigned int>(n - 1);
                    }
                    __syncthreads();
                    if (*last == 0) break;
                    // common max and sum by row, 8 or 16 threads to a row; then the pieces' weights
                    float* wts = merge;  // [8][kRowsMax]
                    {
                        constexpr int kPer = kDecodeThreads / kRows;
                        const int r = threadIdx.x / kPer, sub = threadIdx.x % kPer;
                        float mk = -INFINITY, lk = 0.0f;
                        if (sub < n) {
                            mk = __ldcg(piece(sub) + kRows * D + r);
                            lk = __ldcg(piece(sub) + kRows * D + kRows + r);
                        }
                        float mr = mk;
#pragma unroll
                        for (int off = 4; off > 0; off >>= 1) mr = fmaxf(mr, __shfl_xor_sync(0xffffffffu, mr, off));
                        const float w = mk == -INFINITY ? 0.0f : ptx::ex2(mk - mr);
                        lk *= w;
#pragma unroll
                        for (int off = 4; off > 0; off >>= 1) lk += __shfl_xor_sync(0xffffffffu, lk, off);
                        if (sub < 8) wts[sub * kRowsMax + r] = w;
                        if (sub == 0) {
                            stat_m[r] = mr;
                            stat_l[r] = lk;
                        }
                    }
                    __syncthreads();
                    // O in float4 units of the rows, two to a thread
                    const int units = rows * (D / 4);
#pragma unroll 1
                    for (int u0 = threadIdx.x; u0 < units; u0 += 2 * kDecodeThreads) {
                        const int u1 = u0 + kDecodeThreads;
                        float4 y0[8], y1[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float4* pk = reinterpret_cast<const float4*>(piece(min(k, n - 1)));
                            y0[k] = __ldcg(pk + u0);
                            y1[k] = u1 < units ? __ldcg(pk + u1) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        }
                        const int r0 = u0 / (D / 4), r1 = min(u1, units - 1) / (D / 4);
                        float4 x0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), x1 = x0;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float w0 = k < n ? wts[k * kRowsMax + r0] : 0.0f;
                            const float w1 = k < n ? wts[k * kRowsMax + r1] : 0.0f;
                            x0.x += w0 * y0[k].x;
                            x0.y += w0 * y0[k].y;
                            x0.z += w0 * y0[k].z;
                            x0.w += w0 * y0[k].w;
                            x1.x += w1 * y1[k].x;
                            x1.y += w1 * y1[k].y;
                            x1.z += w1 * y1[k].z;
                            x1.w += w1 * y1[k].w;
                        }
                        if (pieces <= 8) {
                            write_out(r0, (u0 % (D / 4)) * 4, x0, stat_l[r0]);
                            if (u1 < units) write_out(r1, (u1 % (D / 4)) * 4, x1, stat_l[r1]);
                        } else {
                            reinterpret_cast<float4*>(group)[u0] = x0;
                            if (u1 < units) reinterpret_cast<float4*>(group)[u1] = x1;
                        }
                    }
                    if (threadIdx.x < rows) {
                        if (pieces <= 8) {
                            write_lse(threadIdx.x, stat_m[threadIdx.x], stat_l[threadIdx.x]);
                        } else {
                            group[kRows * D + threadIdx.x] = stat_m[threadIdx.x];
                            group[kRows * D + kRows + threadIdx.x] = stat_l[threadIdx.x];
                        }
                    }
                }
                if (pieces <= 8) break;
                counter += kDecodeMaxCtas;  // a row of counters per level
                index >>= 3;
                pieces = (pieces + 7) >> 3;
                stride <<= 3;
            }
            __syncthreads();  // before the next piece writes what was read here
        }
        item0 += cur.n + kItemCost;
        if (!cur.next(a)) break;
    }
    cp_async_wait<0>();
}

// ------------------------------------------------------------------------------ append
//
// A copy with a gather of page ids: each new row is read once and written once.  Threads take 16 bytes of a K row
// and the same of the V row; a block takes kAppendRows rows of (sequence, kv-head, token), the token
// fastest, which is the order of both sides, and issues all of its loads before its first store.
constexpr int kAppendThreads = 256;
constexpr int kAppendUnroll = 4;  // rows of a thread, where that still makes a block for every SM

// A scale as the append kernel divides by it: two factors whose products with a value lie on either side of
// the fp32 quotient (and are the quotient for a power of two).
struct Divisor {
    float scale, lo, hi;
    bool bracket;  // the reciprocal is a normal number
    __device__ __forceinline__ explicit Divisor(float s) : scale(s) {
        const uint32_t u = __float_as_uint(s);
        const uint32_t e = u >> 23;  // positive scales only (a sign makes e large)
        bracket = e > 7 && e < 247;
        const float inv = 1.0f / s;
        const bool exact = (u & 0x7fffffu) == 0;
        lo = exact ? inv : inv * (1.0f - 0x1p-21f);
        hi = exact ? inv : inv * (1.0f + 0x1p-21f);
    }
};

// Four values (two pairs) to e4m3, the first in the lowest byte.
__device__ __forceinline__ uint32_t e4m3x4(uint64_t ab, uint64_t cd) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(ptx::lo_f32(ab)), "f"(ptx::hi_f32(ab)), "f"(ptx::lo_f32(cd)), "f"(ptx::hi_f32(cd)));
    return r;
}

// Eight bf16 values over a scale, to nearest e4m3 (ties to even), saturated; NaN stays.  Rounding is
// monotonic, so where the two products round to one e4m3 value the quotient between them does too; where
// they do not (a quotient within 2^-21 of the middle of two values, about one in 10^5), it is divided.
// On 100 MB of new rows, whose bytes take 23 us at the copy rate, that takes 37, dividing all of them 53.
__device__ __forceinline__ uint2 quantise8(uint4 w, const Divisor& d) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    const uint64_t lo2 = ptx::f32x2(d.lo), hi2 = ptx::f32x2(d.hi);
    uint64_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = ptx::f32x2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xFFFF0000u));
    uint2 lo, hi;
    lo.x = e4m3x4(ptx::fmul2(x[0], lo2), ptx::fmul2(x[1], lo2));
    hi.x = e4m3x4(ptx::fmul2(x[0], hi2), ptx::fmul2(x[1], hi2));
    lo.y = e4m3x4(ptx::fmul2(x[2], lo2), ptx::fmul2(x[3], lo2));
    hi.y = e4m3x4(ptx::fmul2(x[2], hi2), ptx::fmul2(x[3], hi2));
    if (!d.bracket || lo.x != hi.x || lo.y != hi.y) {
        auto over = [&](uint64_t p) { return ptx::f32x2(ptx::lo_f32(p) / d.scale, ptx::hi_f32(p) / d.scale); };
        lo.x = e4m3x4(over(x[0]), over(x[1]));
        lo.y = e4m3x4(over(x[2]), over(x[3]));
    }
    return lo;
}

template <int D, bool kE4M3, int kUnroll>
__global__ void __launch_bounds__(kAppendThreads, 4) paged_append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int kVecs = D / 8;                        // threads of a row
    constexpr int kRowsPer = kAppendThreads / kVecs;    // rows of a block at a time
    const int c = threadIdx.x % kVecs;
    const uint32_t rows = static_cast<uint32_t>(a.batch) * a.tokens * a.c.heads_kv;
    const uint32_t row0 = blockIdx.x * (kRowsPer * kUnroll) + threadIdx.x / kVecs;
    // three steps, each with the loads of all rows side by side: starts and counts, then page ids and
    // the new rows, then the stores
    int b[kUnroll], h[kUnroll], t[kUnroll], start[kUnroll], count[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const uint32_t row = row0 + i * kRowsPer;
        const uint32_t bh = fast_div(min(row, rows - 1), a.fd_tokens);
        t[i] = static_cast<int>(min(row, rows - 1) - bh * a.fd_tokens.d);
        b[i] = static_cast<int>(fast_div(bh, a.fd_heads));
        h[i] = static_cast<int>(bh) - b[i] * a.c.heads_kv;
        start[i] = __ldg(a.starts + b[i]);
        count[i] = a.counts ? __ldg(a.counts + b[i]) : a.tokens;
        if (row >= rows) count[i] = 0;
    }
    int page[kUnroll], slot[kUnroll];
    uint4 kx[kUnroll], vx[kUnroll];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        bool ok = t[i] < count[i];
        const int64_t pos = static_cast<int64_t>(start[i]) + t[i];
        if (pos < 0 || pos >= static_cast<int64_t>(a.c.max_pages) * a.c.page_size) {
            bad |= ok;
            ok = false;
        }
        const int at = static_cast<int>(fast_div(static_cast<uint32_t>(pos), a.c.fd_page));
        slot[i] = ok ? static_cast<int>(pos) - at * a.c.page_size : -1;
        page[i] = ok ? __ldg(a.c.table + b[i] * a.c.table_stride + at) : 0;
        const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(a.k) + b[i] * a.k_b + h[i] * a.k_h + t[i] * a.k_t;
        const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v) + b[i] * a.v_b + h[i] * a.v_h + t[i] * a.v_t;
        if (ok) kx[i] = __ldg(reinterpret_cast<const uint4*>(k) + c);
        if (ok) vx[i] = __ldg(reinterpret_cast<const uint4*>(v) + c);
    }
    // the divisors of the first row's head, which most often is every row's
    Divisor kd(1.0f), vd(1.0f);
    int held = -1;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        if (slot[i] < 0) continue;
        if (page[i] < 0 || page[i] >= a.c.num_pages) {
            bad = true;
            continue;
        }
        uint8_t* k = a.c.k + page[i] * a.c.k_page + h[i] * a.c.k_head + slot[i] * a.c.k_slot;
        uint8_t* v = a.c.v + page[i] * a.c.v_page + h[i] * a.c.v_head + slot[i] * a.c.v_slot;
        if constexpr (kE4M3) {
            if (h[i] != held) {
                held = h[i];
                kd = Divisor(a.c.k_scale ? __ldg(a.c.k_scale + held) : 1.0f);
                vd = Divisor(a.c.v_scale ? __ldg(a.c.v_scale + held) : 1.0f);
            }
            reinterpret_cast<uint2*>(k)[c] = quantise8(kx[i], kd);
            reinterpret_cast<uint2*>(v)[c] = quantise8(vx[i], vd);
        } else {
            reinterpret_cast<uint4*>(k)[c] = kx[i];
            reinterpret_cast<uint4*>(v)[c] = vx[i];
        }
    }
    if (bad) bad_page(a.c);
}

// ------------------------------------------------------------------------------ page copy
//
// Pairs travel in the launch's parameters.  A block copies kCopyBytes of a page's K or V in one layer, all of
// its loads before its first store.
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 8;
constexpr int64_t kCopyBytes = kCopyThreads * kCopyUnroll * 16;
constexpr int kPairsFew = 16, kPairsMany = 400;  // pairs of a launch

template <int N>
struct PairList {
    int32_t id[2 * N];
};

template <int N>
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const __grid_constant__ CopyArgs a,
                                                                 const __grid_constant__ PairList<N> list) {
    const int which = blockIdx.z & 1;
    const int layer = blockIdx.z >> 1;
    const int pair = blockIdx.y;
    uint8_t* base = a.base[which] + layer * a.layer[which];
    const uint8_t* src = base + list.id[2 * pair] * a.page[which];
    uint8_t* dst = base + list.id[2 * pair + 1] * a.page[which];
    const int64_t vecs = a.run_bytes[which] / 16;
    const int64_t total = vecs * a.inner[which] * a.outer[which];
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kCopyThreads * kCopyUnroll) + threadIdx.x;
    if (total == vecs) {  // the page is one run of bytes
        uint4 x[kCopyUnroll];
#pragma unroll
        for (int i = 0; i < kCopyUnroll; ++i)
            if (first + i * kCopyThreads < total) x[i] = __ldcs(reinterpret_cast<const uint4*>(src) + first + i * kCopyThreads);
#pragma unroll
        for (int i = 0; i < kCopyUnroll; ++i)
            if (first + i * kCopyThreads < total) __stcs(reinterpret_cast<uint4*>(dst) + first + i * kCopyThreads, x[i]);
        return;
    }
#pragma unroll 4
    for (int i = 0; i < kCopyUnroll; ++i) {
        const int64_t at = first + i * kCopyThreads;
        if (at < total) {
            const int64_t run = at / vecs;
            const int64_t o = run / a.inner[which];
            const int64_t off = o * a.outer_stride[which] + (run - o * a.inner[which]) * a.inner_stride[which] + (at - run * vecs) * 16;
            *reinterpret_cast<uint4*>(dst + off) = __ldg(reinterpret_cast<const uint4*>(src + off));
        }
    }
}

template <int N>
cudaError_t launch_copy(const CopyArgs& a, int64_t first, int64_t count, cudaStream_t stream) {
    PairList<N> list;
    for (int64_t i = 0; i < 2 * count; ++i) list.id[i] = a.pairs[2 * first + i];
    int64_t bytes = 0;
    for (int w = 0; w < 2; ++w) bytes = std::max(bytes, a.run_bytes[w] * a.inner[w] * a.outer[w]);
    const int64_t blocks = (bytes + kCopyBytes - 1) / kCopyBytes;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    constexpr int kLayers = 32767;  // of a launch
    for (int l = 0; l < a.layers; l += kLayers) {
        CopyArgs x = a;
        x.pairs = nullptr;
        x.layers = std::min(a.layers - l, kLayers);
        for (int w = 0; w < 2; ++w) x.base[w] += l * x.layer[w];
        const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(count), 2 * x.layers);
        page_copy_kernel<N><<<grid, kCopyThreads, 0, stream>>>(x, list);
    }
    return cudaGetLastError();
}

}  // namespace

size_t decode_workspace_bytes(int32_t head_dim) {
    return kDecodeCounterBytes + 2 * sizeof(float) * kDecodeMaxCtas * (static_cast<size_t>(kRowsMax) * head_dim + 2 * kRowsMax);
}

namespace {

// Most keys that a sequence of this call can have visible.
int64_t decode_keys(const DecodeArgs& a) {
    const int64_t room = static_cast<int64_t>(a.c.max_pages) * a.c.page_size;
    return a.window > 0 ? std::min<int64_t>(room, static_cast<int64_t>(a.window) + a.sinks) : room;
}

template <int D, bool kE4M3, int R>
cudaError_t launch_decode(DecodeArgs& a, cudaStream_t stream) {
    using Cfg = DecodeCfg<D, kE4M3, R>;
    a.row_tiles = (a.group + Cfg::kRows - 1) / Cfg::kRows;
    a.items_per_seq = a.c.heads_kv * a.row_tiles;
    a.fd_items = make_fastdiv(static_cast<uint32_t>(a.items_per_seq));
    // no more CTAs than the page table's room could give work to, but one for every piece of few items
    const int64_t keys = decode_keys(a);
    const int64_t items = static_cast<int64_t>(a.items_per_seq) * a.batch;
    const int64_t slices = (keys + Cfg::kSlice - 1) / Cfg::kSlice;
    const int64_t worth = std::max((slices + kMinSlices - 1) / kMinSlices, static_cast<int64_t>(kFewItems)) * items;
    const int64_t most = std::min<int64_t>(Cfg::kCtas * 148, static_cast<int64_t>(Cfg::kCtas) * a.sm_count);
    const unsigned grid = static_cast<unsigned>(std::min(most, worth));
    paged_decode_kernel<D, kE4M3, R><<<grid, kDecodeThreads, Cfg::kSmemBytes, stream>>>(a);
    return cudaGetLastError();
}

template <int D, bool kE4M3>
cudaError_t launch_decode(DecodeArgs& a, cudaStream_t stream) {
    return a.group <= 8 ? launch_decode<D, kE4M3, 1>(a, stream) : launch_decode<D, kE4M3, 2>(a, stream);
}

template <int D, bool kE4M3, int R>
int64_t decode_work(const DecodeArgs& a) {
    using Cfg = DecodeCfg<D, kE4M3, R>;
    const int64_t items = static_cast<int64_t>(a.batch) * a.c.heads_kv * ((a.group + Cfg::kRows - 1) / Cfg::kRows);
    return ((decode_keys(a) + Cfg::kSlice - 1) / Cfg::kSlice + kItemCost) * items;
}

}  // namespace

bool decode_work_fits(const DecodeArgs& a, int32_t head_dim, int32_t kv_dtype) {
    auto work = [&](auto one, auto two) { return a.group <= 8 ? one(a) : two(a); };
    int64_t n;
    if (kv_dtype == ODF_DTYPE_E4M3)
        n = head_dim == 64 ? work(decode_work<64, true, 1>, decode_work<64, true, 2>)
                           : work(decode_work<128, true, 1>, decode_work<128, true, 2>);
    else
        n = head_dim == 64 ? work(decode_work<64, false, 1>, decode_work<64, false, 2>)
                           : work(decode_work<128, false, 1>, decode_work<128, false, 2>);
    return n <= 0x7fffffffLL;
}

cudaError_t set_paged_kernel_attrs() {
    auto set = [](auto kernel, int bytes) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    cudaError_t e = set(paged_decode_kernel<64, false, 1>, DecodeCfg<64, false, 1>::kSmemBytes);
    if (e == cudaSuccess) e = set(paged_decode_kernel<64, false, 2>, DecodeCfg<64, false, 2>::kSmemBytes);
    if (e == cudaSuccess) e = set(paged_decode_kernel<128, false, 1>, DecodeCfg<128, false, 1>::kSmemBytes);
    if (e == cudaSuccess) e = set(paged_decode_kernel<128, false, 2>, DecodeCfg<128, false, 2>::kSmemBytes);
    if (e == cudaSuccess) e = set(paged_decode_kernel<64, true, 1>, DecodeCfg<64, true, 1>::kSmemBytes);
    if (e == cudaSuccess) e = set(paged_decode_kernel<64, true, 2>, DecodeCfg<64, true, 2>::kSmemBytes);
    if (e == cudaSuccess) e = set(paged_decode_kernel<128, true, 1>, DecodeCfg<128, true, 1>::kSmemBytes);
    if (e == cudaSuccess) e = set(paged_decode_kernel<128, true, 2>, DecodeCfg<128, true, 2>::kSmemBytes);
    return e;
}

int launch_paged_decode(DecodeArgs& a, int32_t head_dim, int32_t kv_dtype, cudaStream_t stream, const char** err) {
    static_assert(kDecodeCounterBytes >= 3 * kDecodeMaxCtas * sizeof(unsigned int), "three counters per CTA");
    static_assert(kDecodeMaxCtas <= 512, "three levels of eights");
    a.k16_page = static_cast<uint32_t>(a.c.k_page / 16);
    a.k16_head = static_cast<uint32_t>(a.c.k_head / 16);
    a.k16_slot = static_cast<uint32_t>(a.c.k_slot / 16);
    a.v16_page = static_cast<uint32_t>(a.c.v_page / 16);
    a.v16_head = static_cast<uint32_t>(a.c.v_head / 16);
    a.v16_slot = static_cast<uint32_t>(a.c.v_slot / 16);
    cudaError_t e;
    if (kv_dtype == ODF_DTYPE_E4M3)
        e = head_dim == 64 ? launch_decode<64, true>(a, stream) : launch_decode<128, true>(a, stream);
    else
        e = head_dim == 64 ? launch_decode<64, false>(a, stream) : launch_decode<128, false>(a, stream);
    if (e == cudaSuccess) return ODF_OK;
    *err = cudaGetErrorString(e);
    return ODF_ERR_CUDA;
}

namespace {

template <int D, bool kE4M3>
void launch_append(const AppendArgs& a, int64_t rows, cudaStream_t stream) {
    constexpr int64_t kRowsPer = kAppendThreads / (D / 8);
    const int64_t wide = (rows + kRowsPer * kAppendUnroll - 1) / (kRowsPer * kAppendUnroll);
    if (wide >= a.sm_count)
        paged_append_kernel<D, kE4M3, kAppendUnroll><<<static_cast<unsigned>(wide), kAppendThreads, 0, stream>>>(a);
    else
        paged_append_kernel<D, kE4M3, 1>
            <<<static_cast<unsigned>((rows + kRowsPer - 1) / kRowsPer), kAppendThreads, 0, stream>>>(a);
}

}  // namespace

int launch_paged_append(AppendArgs& a, int32_t head_dim, int32_t kv_dtype, cudaStream_t stream, const char** err) {
    const bool e4m3 = kv_dtype == ODF_DTYPE_E4M3;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.tokens * a.c.heads_kv;
    if (rows > 0x7fffffffLL) {
        *err = "batch x kv-heads x tokens is beyond the kernel's 32 bits";
        return ODF_ERR_UNSUPPORTED;
    }
    a.fd_tokens = make_fastdiv(static_cast<uint32_t>(a.tokens));
    a.fd_heads = make_fastdiv(static_cast<uint32_t>(a.c.heads_kv));
    if (head_dim == 64) {
        if (e4m3)
            launch_append<64, true>(a, rows, stream);
        else
            launch_append<64, false>(a, rows, stream);
    } else {
        if (e4m3)
            launch_append<128, true>(a, rows, stream);
        else
            launch_append<128, false>(a, rows, stream);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) *err = cudaGetErrorString(e);
    return e == cudaSuccess ? ODF_OK : ODF_ERR_CUDA;
}

int launch_page_copy(const CopyArgs& a, cudaStream_t stream, const char** err) {
    cudaError_t e = cudaSuccess;
    for (int64_t first = 0; first < a.n_pairs && e == cudaSuccess;) {
        const int64_t count = std::min<int64_t>(a.n_pairs - first, kPairsMany);
        e = count <= kPairsFew ? launch_copy<kPairsFew>(a, first, count, stream) : launch_copy<kPairsMany>(a, first, count, stream);
        first += count;
    }
    if (e != cudaSuccess) *err = cudaGetErrorString(e);
    return e == cudaSuccess ? ODF_OK : ODF_ERR_CUDA;
}

}  // namespace odf
