// Attention of new tokens' queries over a paged cache, 16-bit or 4-bit: out = softmax(scale q k^T + mask) v.
//
// What bounds it: reading the cached rows once.  A KV head's queries (count tokens x G heads, 8, 16 or 32 rows at a time)
// share every row that is read, and the products run on mma.sync (m16n8k16): a step of generation needs a few rows of
// a product, where tcgen05's 128 would be padding, and its operands come straight from the registers that decode 4 bits.
//
// Up to 16 rows at a time, queries and probabilities go through the products in two 16-bit parts each (the value rounded, and what
// the rounding left), so that only the result is rounded to 16 bits.  With up to 8 rows the second parts are rows 8 ... 15 of
// the same product, which would be padding, and cost nothing; with up to 16 they are a second product.
//
// Every warp is a stream of its own: it copies blocks of KB keys into its ring in shared memory (cp.async, NST - 1 blocks
// ahead, also across the ends of its work), waits for its own copies only, and keeps its own running maximum, sum and
// accumulator in registers; there is no barrier in the loop.  Rows outside the item's key range are filled with zeros and
// not read, so nothing that lies there can reach a result.
//
// Work: the blocks of all (sequence, KV head, row group) items form one line, cut evenly between the CTAs whatever the
// lengths are; the four warps of a CTA take a segment's blocks in turn and add up through their free ring slots.
// An item inside one CTA is finished there; parts of a divided one are parked and added in the order of the CTAs by
// combine_kernel, so results do not depend on which CTA finishes first.  The host needs no lengths for any of this.
//
// Measured (replayed in a graph), heads 32/8 of 128 elements, one token: 64 sequences of up to 8192 keys in 16 bits 211 us (6.5 TB/s, what
// a copy reaches); 16 of up to 16,384 in 4 bits 72 us (2.75 TB/s: 795 instructions a warp and 32 keys, at 12 warps per SM); one sequence
// of 500 keys 8.5 us (latency).
#pragma once

#include "cache.cuh"

namespace bob {

struct alignas(16) PagedParams {
    bob_sm100_rotary rotary;      // pairs 0: queries are taken as they are
    SequenceParams seq;
    CacheTensor cache[2];
    const uint16_t* q; long long q_sb, q_sh, q_sn;
    uint16_t* out;                // contiguous [B, Hq, N, D]
    int Hq, Hkv, G, N, form;
    int g_part;                   // 65536 / G + 1: x / G = x * g_part / 65536 for the x of an item's rows, below 64, and G up to 32
    int groups;                   // row groups of ROWS query rows per KV head
    int causal, window;
    int alike;                    // keys and values (and their scales) have the same strides
    float scale;
    float* part_ml;               // [CTAs][2][ROWS] (reference, sum)
    float* part_acc;              // [CTAs][2][ROWS][D]
    int ctas;                     // CTAs of paged_kernel
};

constexpr float kLog2e = 1.4426950408889634f, kNone = -3e38f;         // (kNone: the reference of a row without keys)
constexpr int kPagedWarps = 4, kPagedThreads = 32 * kPagedWarps;
constexpr int kPagedMinBlocks = 4;          // blocks that are worth a CTA of their own
constexpr int kLevel = 8;                   // a warp's blocks between two levellings of 4-bit values' sums (16 or 32 products' steps)

template <int D_, int ROWS_, int BITS_>
struct PagedConfig {
    static constexpr int D = D_, ROWS = ROWS_, BITS = BITS_;
    static constexpr bool PARTS = ROWS <= 16;                    // two parts of queries and probabilities
    static constexpr int MT = ROWS == 8 ? 1 : 2;                 // products of 16 rows
    static constexpr int LR = ROWS / 8;                          // rows of a thread
    // 16 bits: 4 KB of keys and 4 KB of values per block.  4 bits: 2 to 2.5 KB each, where the work per block counts.
    static constexpr int KB = BITS == 16 ? 2048 / D : (D == 128 ? 32 : 64);
    static constexpr int SUB = BITS == 16 ? KB : 32;             // keys of a block that are computed at a time
    static_assert(KB % SUB == 0 && SUB % 16 == 0, "whole products");
    static constexpr int ROW_BYTES = D * BITS / 8, CHUNKS = ROW_BYTES / 16;
    // 4 bits: a thread reads a word of four rows two apart; these strides put the rows into different banks
    static constexpr int V_STRIDE = BITS == 16 ? ROW_BYTES : (D == 128 ? 80 : (D == 64 ? 48 : 16));
    static constexpr int OFF_V = KB * ROW_BYTES, OFF_SK = OFF_V + KB * V_STRIDE, OFF_SV = OFF_SK + (BITS == 4 ? KB * 8 : 0);
    static constexpr int STAGE = OFF_SV + (BITS == 4 ? KB * 8 : 0);
    static constexpr int CTAS = ROWS == 8 ? 3 : 2;
    static constexpr int NST = BITS == 16 ? (CTAS == 2 ? 3 : 2) : (CTAS == 2 ? 4 : 3);
    // columns that EX_ROWS rows of an accumulator bring into a ring slot at a time
    static constexpr int EX_ROWS = ROWS == 8 ? 8 : 16;
    static constexpr int EX_COLS = 4 * EX_ROWS * D <= STAGE ? D : D / 2;
    static_assert(4 * EX_ROWS * EX_COLS <= STAGE && STAGE % 16 == 0, "an accumulator passes through a slot");
    static constexpr int Q_STRIDE = 2 * D + 16;                  // bytes of a query row; the 16 spread rows over the banks
    static constexpr int OFF_Q = kPagedWarps * NST * STAGE, OFF_ML = OFF_Q + 16 * MT * Q_STRIDE;
    static constexpr int OFF_SLOT = OFF_ML + 2 * kPagedWarps * EX_ROWS * 4;
    static constexpr int OFF_QF = OFF_SLOT + 16;                 // 4 bits: queries as the products' operands, [product][step][lane]
    static constexpr int SMEM = OFF_QF + (BITS == 4 ? MT * (D / 16) * 512 : 0);
    static_assert(OFF_QF % 16 == 0, "16-byte loads");
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(there ? 8 : 0) : "memory");
}
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int WORDS> __device__ __forceinline__ void lds_words(uint32_t addr, uint32_t* w) {
    if constexpr (WORDS == 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
    else if constexpr (WORDS == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A factor that neither infinities nor zeros are lost on.
__device__ __forceinline__ float in_range(float x) { return fminf(fmaxf(x, 0x1p-126f), 3e38f); }

// x 2^n for |n| up to 252, in two steps: 2^n alone may be no fp32 number.
__device__ __forceinline__ float power_of_two(int n) { return __uint_as_float(static_cast<uint32_t>(127 + n) << 23); }
__device__ __forceinline__ float times_power(float x, int n) { return x * power_of_two(n / 2) * power_of_two(n - n / 2); }

// A product with a value's first part, and with the rest of it.  An infinite element makes the second one infinite of
// either sign or NaN, and decides the first alone.
// (Codes are finite.)
template <int BITS>
__device__ __forceinline__ float whole(float first, float rest) { return BITS == 4 || fabsf(rest) < INFINITY ? first + rest : first; }

// Pairs of codes (nibbles i and i + 4 of a word) as pairs of fp16 numbers: one logic operation, and a shift for two of them.
// The bits of c alone are the subnormal number c 2^-24 (i even) or c 2^-20 (i odd).
__device__ __forceinline__ uint32_t subnormal_codes(uint32_t w, int i) { return (i & 2 ? w >> 8 : w) & (i & 1 ? 0x00f000f0u : 0x000f000fu); }

// ... as pairs of bf16 numbers 16 + c: a shift and one logic operation, if mask and exponent come from registers (with both as
// constants the compiler takes two operations).
struct CodePairs {
    uint32_t mask, one;
    __device__ __forceinline__ CodePairs() {
        asm volatile("mov.b32 %0, %1;" : "=r"(mask) : "n"(0x000f000fu << 3));       // the mantissa's upper four bits
        asm volatile("mov.b32 %0, %1;" : "=r"(one) : "n"(0x41804180u));
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t w, int i) const {
        const int by = 4 * i - 3;
        const uint32_t x = by < 0 ? w << -by : w >> by;
        uint32_t r;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(one));       // (x & mask) | one
        return r;
    }
};

// Blocks [first, first + n) of KB keys that the queries of sequence b attend to, of every KV head and row group.
struct BlockRange { int first, n; };
template <int KB>
__device__ __forceinline__ BlockRange blocks_of(const PagedParams& p, int b) {
    const Sequence s = sequence_of(p.seq, b, p.N);
    int lo = 0;
    if (p.window > 0) lo = max(0, s.start - p.window + 1);
    if (s.count == 0 || s.length <= lo) return {0, 0};
    const int first = lo / KB;
    return {first, (s.length + KB - 1) / KB - first};
}

__device__ __forceinline__ long long quotient(long long a, long long b) {       // both not negative; 32 bits where they do
    return (a | b) >> 32 ? a / b : static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
}

// The line of all blocks, and where it is cut: into stretches of equal length, one for each CTA.  With fewer items than CTAs
// and little work every item is cut into the same number of stretches, so that none has parts of two items (their queries,
// sums and parts to add cost as much as a few blocks: 128 items of 33 blocks 17.6 us without, 14.8 with).
struct Line {
    long long total, base;        // blocks; blocks of a stretch, the first `rest` have one more
    int parts, rest, lane_n;
    // lane_n: the blocks of sequence `lane` (of the first 32)
    template <int KB>
    __device__ __forceinline__ void measure(const PagedParams& p, int lane) {
        lane_n = lane < p.seq.B ? blocks_of<KB>(p, lane).n : 0;
        long long sum = lane_n;
        int items = lane_n > 0;
        for (int b = lane + 32; b < p.seq.B; b += 32) {
            const int n = blocks_of<KB>(p, b).n;
            sum += n;
            items += n > 0;
        }
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            items += __shfl_xor_sync(0xffffffffu, items, o);
        }
        const long long per = p.Hkv * p.groups;
        total = sum * per;
        parts = static_cast<int>(min((long long)p.ctas, max(1LL, total / kPagedMinBlocks)));
        if (total > 0 && items * per <= parts && total < 32LL * parts) {
            const int whole = static_cast<int>(items * per), equal = parts / whole * whole;
            if (5 * equal >= 4 * parts) parts = equal;
        }
        base = quotient(total, parts);
        rest = static_cast<int>(total - base * parts);
    }
    __device__ __forceinline__ long long cut(int i) const { return base * i + min(i, rest); }
    // the stretch that block `at` lies in
    __device__ __forceinline__ int stretch(long long at) const {
        const long long longer = (base + 1) * rest;
        return static_cast<int>(at < longer ? quotient(at, base + 1) : rest + quotient(at - longer, max(1LL, base)));
    }
};

// Walks the items of a CTA's stretch of the line.
template <int KB>
struct Cursor {
    long long pos, end, base;     // base: where sequence b begins on the line
    int b, first, n;              // its blocks
    // the segment: blocks [blk, last) of an item, reduced to those that its rows attend to
    int kv_head, group, blk, last, lo, hi;
    bool whole, begins;           // the segment is the whole item; ... has its first block

    // Finds the sequence that a stretch begins in.
    __device__ __forceinline__ void start(const PagedParams& p, const Line& line, int part, int lane) {
        pos = line.cut(part); end = line.cut(part + 1); base = 0; b = 0; first = 0; n = 0;
        if (pos >= end) return;
        const int per = p.Hkv * p.groups;
        for (int b0 = 0;; b0 += 32) {
            const int mine = b0 == 0 ? line.lane_n : (b0 + lane < p.seq.B ? blocks_of<KB>(p, b0 + lane).n : 0);
            int upto = mine;
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += t;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, base + (long long)upto * per > pos);
            if (past || b0 + 32 >= p.seq.B) {
                const int l = past ? __ffs(past) - 1 : 31;
                b = b0 + l;
                base += (long long)__shfl_sync(0xffffffffu, upto - mine, l) * per;
                break;
            }
            base += (long long)__shfl_sync(0xffffffffu, upto, 31) * per;
        }
        const BlockRange r = blocks_of<KB>(p, b);
        first = r.first; n = r.n;
    }
    // The next segment; false at the end.
    template <int ROWS>
    __device__ __forceinline__ bool next(const PagedParams& p) {
        if (pos >= end) return false;
        const int per = p.Hkv * p.groups;
        while (pos >= base + (long long)n * per) {
            base += (long long)n * per;
            const BlockRange r = blocks_of<KB>(p, ++b);
            first = r.first; n = r.n;
        }
        const int at = static_cast<int>(pos - base), item = at / n, off = at - item * n;
        const int take = static_cast<int>(min((long long)(n - off), end - pos));
        kv_head = item;
        group = 0;
        if (p.groups > 1) {
            kv_head = item / p.groups;
            group = item - kv_head * p.groups;
        }
        blk = first + off;
        last = blk + take;
        whole = take == n;
        begins = off == 0;
        pos += take;
        const Sequence s = sequence_of(p.seq, b, p.N);
        int i0 = 0, i1 = min(p.N, s.count) - 1;          // its tokens
        if (p.groups > 1) {
            i0 = group * ROWS / p.G;
            i1 = min(i1, (min((group + 1) * ROWS, p.N * p.G) - 1) / p.G);
        }
        lo = p.window > 0 ? max(0, s.start + i0 - p.window + 1) : 0;
        hi = i0 > i1 ? 0 : (p.causal ? min(s.length, s.start + i1 + 1) : s.length);
        blk = max(blk, lo / KB);
        last = min(last, (hi + KB - 1) / KB);
        return true;
    }
};

// 16 elements of a query row, turned to its position, into shared memory; the second parts go to `rest` (if there).
template <int D, bool BF16, int FORM>
__device__ __forceinline__ void bring_query(const PagedParams& p, uint16_t* dst, uint16_t* rest, const uint16_t* src, int c, int position) {
    const RowPlace<FORM> place(c, p.rotary.pairs);
    Turner<FORM, BF16, float> turn;
    const Chunks x = place.load(src);
    turn.set(p.rotary, c, position);
    float v[16], r[16];
    turn.values(x, v);
    const Chunks y{narrow8<BF16>(v), narrow8<BF16>(v + 8)};
    place.store(dst, y);
    if (!rest) return;
    widen8<BF16>(y.a, r);
    widen8<BF16>(y.b, r + 8);
    #pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = v[i] - r[i];
    place.store(rest, Chunks{narrow8<BF16>(r), narrow8<BF16>(r + 8)});
}

template <int D, int ROWS, bool BF16, int BITS>
__global__ void __launch_bounds__(kPagedThreads, (PagedConfig<D, ROWS, BITS>::CTAS)) paged_kernel(const __grid_constant__ PagedParams p) {
    using CFG = PagedConfig<D, ROWS, BITS>;
    constexpr int KB = CFG::KB, SUB = CFG::SUB, NT = SUB / 8, KS = D / 16, NST = CFG::NST, STAGE = CFG::STAGE, MT = CFG::MT, LR = CFG::LR;
    constexpr bool PARTS = CFG::PARTS;
        extern __shared__ __align__(128) uint8_t paged_smem[];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
    const uint32_t ring = smem_u32(paged_smem) + warp * NST * STAGE;
    constexpr int EXR = CFG::EX_ROWS, EXC = CFG::EX_COLS;
    float* sm_m = reinterpret_cast<float*>(paged_smem + CFG::OFF_ML);            // [warp][EXR]
    float* sm_l = sm_m + kPagedWarps * EXR;
    volatile int* sm_slot = reinterpret_cast<volatile int*>(paged_smem + CFG::OFF_SLOT);
    asm volatile("griddepcontrol.launch_dependents;");

    if (blockIdx.x == 0 && warp == 0) {
        for (int b = lane; b < p.seq.B; b += 32)
            if (!sequence_of(p.seq, b, p.N).ok) report(p.seq.sticky, kStatusBadLength);
    }
    Cursor<KB> src, seg;
    {
        Line line = {};
        line.measure<KB>(p, lane);
        if (static_cast<int>(blockIdx.x) >= line.parts) return;
        src.start(p, line, blockIdx.x, lane);
    }

    // ---- copies: block `blk` of the copying cursor, a warp's every fourth of a segment ----------------------
    seg = src;
    int fill = 0;                                        // ring slot that is free
    bool more = true;
    src.blk = src.last = 0;
    // Lane i: the page of the block's keys 16 i ... if the item reads any of them.  It is asked for a block ahead, and looked
    // at when the block is copied.
    int entry = 0;
    bool asked = false;
    constexpr int RPC = 32 / CFG::CHUNKS;                // rows of a warp-wide copy
    const int copy_row = lane / CFG::CHUNKS, chunk = lane % CFG::CHUNKS;
    auto seek = [&]() {                                  // to this warp's next block, and ask for its pages
        while (more && src.blk >= src.last) {
            more = src.template next<ROWS>(p);
            src.blk += warp;
        }
        if (!more) return;
        const int key = src.blk * KB + 16 * lane;
        asked = lane < KB / 16 && key + 15 >= src.lo && key < src.hi;
        if (asked) entry = page_entry(p.seq, src.b, key);
    };
    auto swizzled = [](int r, int ch) { return BITS == 4 ? ch : ch ^ (CFG::CHUNKS >= 8 ? r & 7 : (r >> 1) & 3); };
    auto copy_block = [&]() {
        if (more) {
            const uint32_t dst = ring + fill * STAGE;
            const int from_lo = src.blk * KB - src.lo, reach = src.hi - src.lo;
            const bool found = asked && static_cast<unsigned>(entry) < static_cast<unsigned>(p.seq.pages);
            if (asked && !found) report(p.seq.sticky, kStatusBadPage);
            const uint32_t pages = __ballot_sync(0xffffffffu, found);
            const int page = found ? entry : 0, row = (src.blk * KB + 16 * lane) & ((1 << p.seq.page_shift) - 1);
            // rows of 16 keys lie in one page, one after another
            auto there = [&](int r) { return static_cast<unsigned>(from_lo + r) < static_cast<unsigned>(reach) && (pages >> (r / 16) & 1); };
            constexpr int STEP = RPC > 16 ? RPC / 16 : 1, GROUPS = KB / 16 / STEP;
            long long at[GROUPS], scale_at[KB / 32 + 1];
            #pragma unroll
            for (int w = 0; w < 2; ++w) {
                const CacheTensor& c = p.cache[w];
                if (w == 0 || !p.alike) {
                    const long long mine = page * c.sp + src.kv_head * c.sh + row * c.sr;
                    #pragma unroll
                    for (int i = 0; i < GROUPS; ++i) at[i] = __shfl_sync(0xffffffffu, mine, i * STEP + copy_row / 16);
                    if constexpr (BITS == 4) {
                        const long long scale = page * c.ssp + src.kv_head * c.ssh + row * c.ssr;
                        #pragma unroll
                        for (int i = 0; i < KB / 32; ++i) scale_at[i] = __shfl_sync(0xffffffffu, scale, 2 * i + lane / 16);
                    }
                }
                #pragma unroll
                for (int i = 0; i < GROUPS; ++i) {
                    const uint8_t* from = c.data + at[i] + (copy_row % 16) * c.sr + 16 * chunk;
                    #pragma unroll
                    for (int k = 0; k < (RPC > 16 ? 1 : 16 / RPC); ++k) {
                        const int r = 16 * i * STEP + copy_row + k * RPC;
                        copy16(dst + (w ? CFG::OFF_V + r * CFG::V_STRIDE : r * CFG::ROW_BYTES) + 16 * swizzled(r, chunk), from + k * RPC * c.sr, there(r));
                    }
                }
                if constexpr (BITS == 4) {
                    #pragma unroll
                    for (int k = 0; k < KB / 32; ++k) {
                        const int r = k * 32 + lane;
                        copy8(dst + (w ? CFG::OFF_SV : CFG::OFF_SK) + 8 * r, c.scales + scale_at[k] + (r % 16) * c.ssr, there(r));
                    }
                }
            }
            src.blk += kPagedWarps;
            seek();
        }
        cp_async_commit();                               // (an empty group at the end keeps the count)
        fill = fill + 1 == NST ? 0 : fill + 1;
    };
    seek();
    #pragma unroll 1
    for (int i = 0; i < NST - 1; ++i) copy_block();
    int slot = 0;                                        // ring slot of the next block to use

    const float c_exp = in_range(p.scale * kLog2e);
    const int R = p.N * p.G;
    const CodePairs value_codes;
    #pragma unroll 1
    while (seg.template next<ROWS>(p)) {
        const Sequence s = sequence_of(p.seq, seg.b, p.N);
        // row r of the item is head (r + skip) % G of token i0 + (r + skip) / G
        const int row0 = seg.group * ROWS, i0 = seg.group ? row0 / p.G : 0, skip = row0 - i0 * p.G;
        auto token_of = [&](int r) { return (r + skip) * p.g_part >> 16; };
        // ---- the item's queries ---------------------------------------------------------------------------
        __syncthreads();                                 // (the last item's are in registers, its sums written)
        #pragma unroll 1
        for (int id = tid; id < ROWS * (D / 16); id += kPagedThreads) {
            const int r = id / (D / 16), c = id % (D / 16), k = token_of(r), i = i0 + k, h = seg.kv_head * p.G + r + skip - k * p.G;
            uint16_t* dst = reinterpret_cast<uint16_t*>(paged_smem + CFG::OFF_Q + (id / (D / 16)) * CFG::Q_STRIDE);
            uint16_t* rest = PARTS ? dst + ROWS * CFG::Q_STRIDE / 2 : nullptr;
            if (row0 + r < R && i < s.count) {
                const uint16_t* from = p.q + seg.b * p.q_sb + h * p.q_sh + i * p.q_sn;
                if (p.form == kHalf) bring_query<D, BF16, kHalf>(p, dst, rest, from, c, s.start + i);
                else if (p.form == kInterleaved) bring_query<D, BF16, kInterleaved>(p, dst, rest, from, c, s.start + i);
                else if (p.form == kQuarter) bring_query<D, BF16, kQuarter>(p, dst, rest, from, c, s.start + i);
                else bring_query<D, BF16, kScattered>(p, dst, rest, from, c, s.start + i);
            } else {
                RowPlace<kInterleaved>(c, 0).store(dst, Chunks{});
                if (PARTS) RowPlace<kInterleaved>(c, 0).store(rest, Chunks{});
            }
        }
        __syncthreads();
        float q_sum[LR];                                 // 4 bits: sum of a row's elements;
        int unit[LR];                                    // its scores are multiples of 2^unit
        (void)q_sum; (void)unit;
        // row of mine (LR of them) that half hr of product mt has, or a part of
        auto my_row = [](int mt, int hr) { return ROWS == 8 ? 0 : ROWS == 16 ? hr : 2 * mt + hr; };
        const uint32_t q_rows = smem_u32(paged_smem) + CFG::OFF_Q, q_frags = smem_u32(paged_smem) + CFG::OFF_QF + 16 * lane;
        if constexpr (BITS == 4) {
            // the elements in the order in which a word of codes yields them: thread t holds words NWD t ... of a
            // key row, and a word's pairs are (e, e + 4).  In fp16, as the codes are, times a power of two that
            // brings the row's largest to 2^14 (a part loses nothing but what is below 2^-38 of it), and those that meet
            // c 2^-20 times 1/16.  Kept in shared memory: the registers that they would take are those of the third CTA per SM.
            constexpr int NWD = D / 32;
            float up[LR];
            #pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                uint32_t frag[KS][4];
                #pragma unroll
                for (int hr = 0; hr < 2; ++hr) {
                    const int k = my_row(mt, hr);
                    const bool rest = PARTS && (ROWS == 8 ? hr : mt) == 1;
                    float f[NWD][8];
                    #pragma unroll
                    for (int j = 0; j < NWD; ++j) {
                        uint32_t w[4];
                        lds_words<4>(q_rows + (mt * 16 + g + 8 * hr) * CFG::Q_STRIDE + 16 * (NWD * t + j), w);
                        widen8<BF16>(make_uint4(w[0], w[1], w[2], w[3]), f[j]);
                    }
                    if (!rest) {
                        float largest = 0.f;
                        #pragma unroll
                        for (int j = 0; j < NWD; ++j) {
                            #pragma unroll
                            for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(f[j][e]));
                        }
                        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                        const int exponent = min(max(static_cast<int>(__float_as_uint(largest) >> 23), 127 - 100), 254);
                        up[k] = __uint_as_float(static_cast<uint32_t>(2 * 127 + 14 - exponent) << 23);
                        unit[k] = exponent - 127 - 14 + 24;
                        q_sum[k] = 0.f;
                    }
                    float sum = 0.f;
                    #pragma unroll
                    for (int j = 0; j < NWD; ++j) {
                        #pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            f[j][e] *= up[k];
                            sum += f[j][e];
                            if (e & 1) f[j][e] *= 0.0625f;
                        }
                        #pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            frag[2 * j + half][hr] = pack2<false>(f[j][2 * half], f[j][2 * half + 4]);
                            frag[2 * j + half][2 + hr] = pack2<false>(f[j][2 * half + 1], f[j][2 * half + 5]);
                        }
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    q_sum[k] = fmaf(sum + __shfl_xor_sync(0xffffffffu, sum, 2), 0x1p-24f, q_sum[k]);
                }
                #pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    if (ks % kPagedWarps == warp) st_shared_v4(q_frags + (mt * KS + ks) * 512, frag[ks][0], frag[ks][1], frag[ks][2], frag[ks][3]);
            }
            __syncthreads();
        }
        auto query = [&](int mt, int ks, uint32_t (&a)[4]) {
            if constexpr (BITS == 16) ldsm4(q_rows + (mt * 16 + lane % 16) * CFG::Q_STRIDE + ks * 32 + (lane / 16) * 16, a);
            else lds_words<4>(q_frags + (mt * KS + ks) * 512, a);
        };
        int lo[LR], hi[LR];                              // keys that my rows attend to
        #pragma unroll
        for (int k = 0; k < LR; ++k) {
            const int i = i0 + token_of(8 * k + g);
            hi[k] = p.causal ? min(s.length, s.start + i + 1) : s.length;
            lo[k] = p.window > 0 ? s.start + i - p.window + 1 : 0;
        }
        // ... that every row of the item does
        const int all_hi = p.causal ? min(s.length, s.start + i0 + 1) : s.length;
        const int all_lo = p.window > 0 ? s.start + i0 + token_of(ROWS - 1) - p.window + 1 : 0;
        // a probability is 2^((x - m) c): the reference m is a score as it is, so that the largest one's difference from it is
        // zero however large both are
        float c[LR];
        #pragma unroll
        for (int k = 0; k < LR; ++k) c[k] = BITS == 4 ? in_range(times_power(c_exp, unit[k])) : c_exp;
        // 4 bits: z: what every column gains; w_sum: the weights that the accumulators' codes have met since the last level()
        float acc[MT][D / 8][4], m[LR], l[LR], z[LR], w_sum[LR];
        #pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            #pragma unroll
            for (int i = 0; i < D / 8; ++i) acc[mt][i][0] = acc[mt][i][1] = acc[mt][i][2] = acc[mt][i][3] = 0.f;
        }
        #pragma unroll
        for (int k = 0; k < LR; ++k) { m[k] = kNone; l[k] = z[k] = w_sum[k] = 0.f; }
        // 4 bits: a code goes through the products as 16 + c, so that an accumulator grows by some 24 times the weights while its
        // result, of values about zero, does not, and the products' sums, which are cut off and not rounded, drift with
        // every step.  So every kLevel blocks, and at a segment's end, what a row's columns have in common, their mean, moves to z
        // together with the offset's share, which it all but cancels: what is left are the columns' differences.
        // (131,072 fp16 keys of like weight in one CTA: off by 4.9e-2 of the result without it, 2.0e-4 with it, one rounding.  8 rows
        // take 1 to 3 % more, 16 and 32 rows of 128 elements 5 to 9 %, for registers.)
        auto level = [&]() {
            #pragma unroll
            for (int k = 0; k < LR; ++k) {
                auto column_sum = [&](int i, int e) -> float& { return acc[PARTS ? 0 : k / 2][i][ROWS == 8 ? e : 2 * (k % 2) + e]; };
                float mean = 0.f, weights = w_sum[k];
                #pragma unroll
                for (int i = 0; i < D / 8; ++i) mean = fmaf(column_sum(i, 0) + column_sum(i, 1), 1.f / D, mean);     // (no sum of columns overflows)
                mean += __shfl_xor_sync(0xffffffffu, mean, 1);
                weights += __shfl_xor_sync(0xffffffffu, weights, 1);
                mean += __shfl_xor_sync(0xffffffffu, mean, 2);
                weights += __shfl_xor_sync(0xffffffffu, weights, 2);
                #pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    column_sum(i, 0) -= mean;
                    column_sum(i, 1) -= mean;
                }
                z[k] = fmaf(0.25f, fmaf(PARTS ? -16.f : -24.f, weights, mean), z[k]);        // (a row's z is the sum of its four threads')
                w_sum[k] = 0.f;
            }
        };
        (void)level;

        #pragma unroll 1
        for (int blk = seg.blk + warp; blk < seg.last; blk += kPagedWarps) {
            copies_wait<NST - 2>();
            __syncwarp();                                // every lane's copies are there, and the free slot is read
            const uint32_t stage = ring + slot * STAGE;
            slot = slot + 1 == NST ? 0 : slot + 1;
            copy_block();

            #pragma unroll 1
            for (int sub = 0; sub < KB / SUB; ++sub) {
            const uint32_t base = stage + sub * SUB * CFG::ROW_BYTES;            // key rows; values, scales:
            const uint32_t base_v = stage + CFG::OFF_V + sub * SUB * CFG::V_STRIDE;
            const uint32_t base_sk = stage + CFG::OFF_SK + sub * SUB * 8, base_sv = stage + CFG::OFF_SV + sub * SUB * 8;
            (void)base_sk; (void)base_sv;
            // ---- scores -----------------------------------------------------------------------------------
            float sc[MT][NT][4], x[LR][NT][2];           // products; scores of my rows
            #pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                #pragma unroll
                for (int i = 0; i < NT; ++i) sc[mt][i][0] = sc[mt][i][1] = sc[mt][i][2] = sc[mt][i][3] = 0.f;
            }
            if constexpr (BITS == 16) {
                #pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint32_t qa[MT][4];
                    #pragma unroll
                    for (int mt = 0; mt < MT; ++mt) query(mt, ks, qa[mt]);
                    #pragma unroll
                    for (int pr = 0; pr < NT / 2; ++pr) {
                        const int r = pr * 16 + (lane / 16) * 8 + lane % 8, ch = 2 * ks + (lane / 8) % 2;
                        uint32_t kf[4];
                        ldsm4(base + r * CFG::ROW_BYTES + 16 * swizzled(r, ch), kf);
                        #pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            mma16816<BF16>(sc[mt][2 * pr], qa[mt], kf[0], kf[1]);
                            mma16816<BF16>(sc[mt][2 * pr + 1], qa[mt], kf[2], kf[3]);
                        }
                    }
                }
            } else {
                // a score is scale q . c + zero sum q, in multiples of the row's unit
                constexpr int NWD = D / 32;
                uint32_t w[NT][NWD];
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt) lds_words<NWD>(base + (8 * nt + g) * CFG::ROW_BYTES + 4 * NWD * t, w[nt]);
                #pragma unroll
                for (int j = 0; j < NWD; ++j) {
                    #pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t qa[MT][4];
                        #pragma unroll
                        for (int mt = 0; mt < MT; ++mt) query(mt, 2 * j + half, qa[mt]);
                        #pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint32_t b0 = subnormal_codes(w[nt][j], 2 * half), b1 = subnormal_codes(w[nt][j], 2 * half + 1);
                            #pragma unroll
                            for (int mt = 0; mt < MT; ++mt) mma16816<false>(sc[mt][nt], qa[mt], b0, b1);
                        }
                    }
                }
            }
            #pragma unroll
            for (int i = 0; i < NT; ++i) {
                uint32_t raw[4];                         // 4 bits: (scale, zero) of keys 2 t and 2 t + 1
                if constexpr (BITS == 4) lds_words<4>(base_sk + 8 * (8 * i + 2 * t), raw);
                #pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if constexpr (ROWS == 8) x[0][i][e] = whole<BITS>(sc[0][i][e], sc[0][i][2 + e]);
                    #pragma unroll
                    for (int hr = 0; hr < 2; ++hr) {
                        if constexpr (ROWS == 16) x[hr][i][e] = whole<BITS>(sc[0][i][2 * hr + e], sc[MT - 1][i][2 * hr + e]);
                        if constexpr (ROWS == 32) { x[hr][i][e] = sc[0][i][2 * hr + e]; x[2 + hr][i][e] = sc[MT - 1][i][2 * hr + e]; }
                    }
                    if constexpr (BITS == 4) {
                        #pragma unroll
                        for (int k = 0; k < LR; ++k) x[k][i][e] = fmaf(x[k][i][e], __uint_as_float(raw[2 * e]), __uint_as_float(raw[2 * e + 1]) * q_sum[k]);
                    }
                }
            }

            // ---- softmax ----------------------------------------------------------------------------------
            const int key0 = blk * KB + sub * SUB;
            const bool masked = key0 < all_lo || key0 + SUB > all_hi;
            if (masked) {
                #pragma unroll
                for (int k = 0; k < LR; ++k) {
                    #pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        #pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int key = key0 + 8 * i + 2 * t + e;
                            if (key < lo[k] || key >= hi[k]) x[k][i][e] = -INFINITY;
                        }
                    }
                }
            }
            uint32_t pa[MT][NT / 2][4];                  // probabilities as the second product's operand
            bool grow = false;
            float top[LR];
            #pragma unroll
            for (int k = 0; k < LR; ++k) {
                float v = fmaxf(x[k][0][0], x[k][0][1]);
                #pragma unroll
                for (int i = 1; i < NT; ++i) v = fmaxf(v, fmaxf(x[k][i][0], x[k][i][1]));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
                top[k] = fmaxf(v, kNone);
                grow = grow || (top[k] - m[k]) * c[k] > 8.f;         // (the scale is positive)
            }
            // the reference moves only when the maximum has outgrown it by 2^8
            if (__any_sync(0xffffffffu, grow)) {
                float f[LR];
                #pragma unroll
                for (int k = 0; k < LR; ++k) {
                    const float ref = fmaxf(m[k], top[k]);
                    f[k] = exp2_ftz((m[k] - ref) * c[k]);
                    m[k] = ref;
                    l[k] *= f[k];
                    if constexpr (BITS == 4) { z[k] *= f[k]; w_sum[k] *= f[k]; }
                }
                #pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    #pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        #pragma unroll
                        for (int e = 0; e < 4; ++e) acc[mt][i][e] *= f[my_row(mt, e >> 1)];
                    }
                }
            }
            #pragma unroll
            for (int i = 0; i < NT; ++i) {
                uint32_t raw[4];                         // 4 bits: (scale, zero) of the values of keys 2 t, 2 t + 1
                if constexpr (BITS == 4) lds_words<4>(base_sv + 8 * (8 * i + 2 * t), raw);
                #pragma unroll
                for (int k = 0; k < LR; ++k) {
                    float pr[2];
                    constexpr bool PB = BITS == 4 || BF16;
                    #pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        pr[e] = exp2_ftz((x[k][i][e] - m[k]) * c[k]);
                        l[k] += pr[e];
                        if constexpr (BITS == 4) {
                            // value = scale b + zero - 16 scale, b = 16 + c: scale b goes through the product, with the scale in
                            // the probability, the rest is the same for every column: the zero goes to z, -16 scale by level().
                            // In bf16 for both types: a scale may lie outside fp16.
                            // (one part: value = scale (b - 24) + zero + 8 scale, where the 24 goes with the rounded weights, so
                            // that their rounding, 2^-9, meets b - 24 and not b)
                            const float scale = __uint_as_float(raw[2 * e]), zero = __uint_as_float(raw[2 * e + 1]);
                            z[k] = fmaf(pr[e], PARTS ? zero : fmaf(8.f, scale, zero), z[k]);
                            pr[e] *= scale;
                            if constexpr (PARTS) w_sum[k] += pr[e];
                        }
                    }
                    const uint32_t first = pack2<PB>(pr[0], pr[1]);
                    float back[2];
                    if constexpr (PB) { back[0] = __uint_as_float(first << 16); back[1] = __uint_as_float(first & 0xffff0000u); }
                    else { const float2 f2 = __half22float2(*reinterpret_cast<const __half2*>(&first)); back[0] = f2.x; back[1] = f2.y; }
                    if constexpr (BITS == 4 && !PARTS) w_sum[k] += back[0] + back[1];
                    if constexpr (PARTS) {
                        const uint32_t rest = pack2<PB>(pr[0] - back[0], pr[1] - back[1]);
                        if constexpr (ROWS == 8) { pa[0][i / 2][2 * (i % 2)] = first; pa[0][i / 2][2 * (i % 2) + 1] = rest; }
                        else { pa[0][i / 2][2 * (i % 2) + k] = first; pa[MT - 1][i / 2][2 * (i % 2) + k] = rest; }
                    } else {
                        pa[k / 2][i / 2][2 * (i % 2) + k % 2] = first;
                    }
                }
            }

            // ---- values -----------------------------------------------------------------------------------
            if constexpr (BITS == 16) {
                #pragma unroll
                for (int kk = 0; kk < NT / 2; ++kk) {
                    #pragma unroll
                    for (int dp = 0; dp < D / 16; ++dp) {
                        const int r = kk * 16 + lane % 16, ch = 2 * dp + lane / 16;
                        uint32_t vf[4];
                        ldsm4_trans(base_v + r * CFG::ROW_BYTES + 16 * swizzled(r, ch), vf);
                        #pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            mma16816<BF16>(acc[mt][2 * dp], pa[mt][kk], vf[0], vf[1]);
                            mma16816<BF16>(acc[mt][2 * dp + 1], pa[mt][kk], vf[2], vf[3]);
                        }
                    }
                }
            } else {
                // thread g holds words NWG g ... of a value row: column n of product (word, nibble) is element
                // 8 (NWG n + word) + nibble.  (D = 32: four words, lanes 4 ... 7 take their upper nibbles.)
                constexpr int NWG = D >= 64 ? D / 64 : 1, NIB = D >= 64 ? 8 : 4;
                #pragma unroll
                for (int kk = 0; kk < NT / 2; ++kk) {
                    uint32_t w[4][NWG];
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = kk * 16 + 2 * t + (k & 1) + 8 * (k >> 1);
                        lds_words<NWG>(base_v + r * CFG::V_STRIDE + 4 * (D >= 64 ? NWG * g : g % 4), w[k]);
                    }
                    #pragma unroll
                    for (int word = 0; word < NWG; ++word) {
                        uint32_t two[2][2];              // [keys 2 t, or 2 t + 8][nibbles 0 ... 3, or 4 ... 7] of two keys
                        #pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            two[k][0] = __byte_perm(w[2 * k][word], w[2 * k + 1][word], 0x5410);
                            two[k][1] = __byte_perm(w[2 * k][word], w[2 * k + 1][word], 0x7632);
                            if (D == 32 && g >= 4) two[k][0] = two[k][1];
                        }
                        #pragma unroll
                        for (int i = 0; i < NIB; ++i) {
                            const uint32_t b0 = value_codes(two[0][i / 4], i % 4), b1 = value_codes(two[1][i / 4], i % 4);
                            #pragma unroll
                            for (int mt = 0; mt < MT; ++mt) mma16816<true>(acc[mt][word * NIB + i], pa[mt][kk], b0, b1);
                        }
                    }
                }
            }
            }   // sub
            if (BITS == 4 && ((blk / kPagedWarps) % kLevel == kLevel - 1 || blk + kPagedWarps >= seg.last)) level();
        }

        // ---- the four warps' parts, through their free ring slots, EXR rows at a time ----------------------
        // the element that column n (0 ... 7) of accumulator tile i stands for
        auto column = [&](int i, int n) {
            if constexpr (BITS == 16) return 8 * i + n;
            else if constexpr (D >= 64) return 8 * ((D / 64) * n + i / 8) + i % 8;
            else return 8 * (n % 4) + 4 * (n / 4) + i;
        };
        __syncwarp();                                    // (the slot that is free now was read last)
        #pragma unroll
        for (int pass = 0; pass < ROWS / EXR; ++pass) {
            if (pass > 0) __syncthreads();
            #pragma unroll
            for (int j = 0; j < EXR / 8; ++j) {
                const int k = pass * (EXR / 8) + j;      // my row
                float sum = l[k], zs = z[k];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if constexpr (BITS == 4) {
                    zs += __shfl_xor_sync(0xffffffffu, zs, 1);
                    z[k] = zs + __shfl_xor_sync(0xffffffffu, zs, 2);
                }
                if (t == 0) { sm_m[warp * EXR + j * 8 + g] = BITS == 4 && m[k] > kNone ? times_power(m[k], unit[k]) : m[k]; sm_l[warp * EXR + j * 8 + g] = sum; }
            }
            if (lane == 0) sm_slot[warp] = (warp * NST + fill) * STAGE;
            #pragma unroll
            for (int part = 0; part < D / EXC; ++part) {
                if (part > 0) __syncthreads();
                float* mine = reinterpret_cast<float*>(paged_smem + (warp * NST + fill) * STAGE);
                #pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    #pragma unroll
                    for (int j = 0; j < EXR / 8; ++j) {
                        #pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int r = g + 8 * j, col = column(i, 2 * t + e) - part * EXC;
                            float v;
                            if constexpr (ROWS == 8) v = whole<BITS>(acc[0][i][e], acc[0][i][2 + e]);
                            else if constexpr (ROWS == 16) v = whole<BITS>(acc[0][i][2 * j + e], acc[MT - 1][i][2 * j + e]);
                            else v = acc[pass][i][2 * j + e];
                            if constexpr (BITS == 4) v += z[pass * (EXR / 8) + j];
                            if (EXC == D || (col >= 0 && col < EXC)) mine[r * EXC + (col ^ ((r & 3) << 3))] = v;
                        }
                    }
                }
                __syncthreads();
                #pragma unroll
                for (int k = 0; k < (EXR * EXC / 4 + kPagedThreads - 1) / kPagedThreads; ++k) {
                    const int id = k * kPagedThreads + tid;
                    const int r = id / (EXC / 4), col = (id % (EXC / 4)) * 4, row = row0 + pass * EXR + r;
                    if (row >= R || (EXR * EXC / 4 < kPagedThreads && id >= EXR * EXC / 4)) continue;
                    float ref = sm_m[r];
                    #pragma unroll
                    for (int w = 1; w < kPagedWarps; ++w) ref = fmaxf(ref, sm_m[w * EXR + r]);
                    float sum = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    #pragma unroll
                    for (int w = 0; w < kPagedWarps; ++w) {
                        const float f = exp2_ftz((sm_m[w * EXR + r] - ref) * c_exp);
                        const float4 x = *reinterpret_cast<const float4*>(paged_smem + sm_slot[w] + 4 * (r * EXC + (col ^ ((r & 3) << 3))));
                        sum = fmaf(f, sm_l[w * EXR + r], sum);
                        v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
                    }
                    const int tk = token_of(pass * EXR + r), i = i0 + tk, h = seg.kv_head * p.G + pass * EXR + r + skip - tk * p.G;
                    if (i >= s.count) sum = 0.f;         // a row behind the sequence's new tokens
                    if (seg.whole) {
                        const float inv = sum == 0.f ? 0.f : 1.f / sum;      // (a row without keys is zero; NaN stays NaN)
                        uint2 o = make_uint2(pack2<BF16>(v.x * inv, v.y * inv), pack2<BF16>(v.z * inv, v.w * inv));
                        if (sum == 0.f) o = make_uint2(0, 0);
                        *reinterpret_cast<uint2*>(p.out + (((long long)seg.b * p.Hq + h) * p.N + i) * D + part * EXC + col) = o;
                    } else {
                        const long long at = (2LL * blockIdx.x + (seg.begins ? 1 : 0)) * ROWS + pass * EXR + r;
                        *reinterpret_cast<float4*>(p.part_acc + at * D + part * EXC + col) = v;
                        if (part == 0 && col == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(ref, sum);
                    }
                }
            }
        }
    }
}

// Adds the parts of a forward whose tiles were divided (SweepParams::splits, pack): one thread per four columns of a row.
template <bool BF16>
__global__ void __launch_bounds__(256) add_splits_kernel(const float* part_ml, const float* part_acc, uint16_t* out, int splits, long long rows, int D, int N, int pack, float scale) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x, row = id / (D / 4);
    const int col = static_cast<int>(id % (D / 4)) * 4;
    if (row >= rows) return;
    const float c_exp = in_range(scale * kLog2e);
    float ref = kNone;
    for (int s = 0; s < splits; ++s) ref = fmaxf(ref, __ldcg(part_ml + 2 * (s * rows + row)));
    float sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    #pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml + 2 * (s * rows + row)));
        const float4 x = __ldcg(reinterpret_cast<const float4*>(part_acc + (s * rows + row) * D + col));
        const float f = exp2_ftz((ml.x - ref) * c_exp);
        sum = fmaf(f, ml.y, sum);
        v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
    }
    const float inv = 1.f / sum;
    uint2 o = make_uint2(pack2<BF16>(v.x * inv, v.y * inv), pack2<BF16>(v.z * inv, v.w * inv));
    if (sum == 0.f) o = make_uint2(0, 0);
    // row (head, i, g) of [B * heads, N, pack]
    const long long head = row / (N * pack);
    const int in = static_cast<int>(row - head * (N * pack)), i = in / pack, g = in - i * pack;
    *reinterpret_cast<uint2*>(out + ((head * pack + g) * N + i) * D + col) = o;
}

// Adds the parts of the items that paged_kernel divided, and writes the zeros of those without keys.  WARPS warps to a query
// row (4, or 1 where there are many rows): D / 4 lanes have a part's columns, and up to 4 * WARPS * 128 / D parts are on
// their way at once.
template <int D, int ROWS, bool BF16, int BITS, int WARPS>
__global__ void __launch_bounds__(kPagedThreads) combine_kernel(const __grid_constant__ PagedParams p) {
    using CFG = PagedConfig<D, ROWS, BITS>;
    constexpr int KB = CFG::KB, LPR = D / 4, PER = 32 / LPR, BATCH = 4, STEP = WARPS * PER;
    __shared__ float2 sm_ml[kPagedWarps * PER];
    __shared__ float4 sm_acc[kPagedWarps * PER][LPR];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, col = (lane % LPR) * 4;
    const int group = warp / WARPS * STEP, mine = (warp % WARPS) * PER + lane / LPR;     // the row's place in shared memory; which of its parts
    const int per = p.Hkv * p.groups, b = blockIdx.x / per, item = blockIdx.x - b * per;
    const int r = blockIdx.y * (kPagedWarps / WARPS) + warp / WARPS, row = (item % p.groups) * ROWS + r;
    const bool row_ok = r < ROWS && row < p.N * p.G;
    // (lengths are inputs: they were there before paged_kernel started)
    Line line = {};
    line.measure<KB>(p, lane);
    long long before = 0;
    for (int i = lane; i < b; i += 32) before += i < 32 ? line.lane_n : blocks_of<KB>(p, i).n;
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    const int n = blocks_of<KB>(p, b).n;
    const long long first = before * per + (long long)item * n;
    int c0 = 0, c1 = 0;                                  // the CTAs that have its blocks
    if (n > 0) {
        c0 = line.stretch(first);
        c1 = line.stretch(first + n - 1);
    }
    // (every CTA waits: this grid must not end, and let the stream go on, before paged_kernel has)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (n > 0 && c0 == c1) return;                       // finished in paged_kernel
    uint16_t* out = p.out + (((long long)b * p.Hq + (item / p.groups) * p.G + row % p.G) * p.N + row / p.G) * D + col;
    if (n == 0) {
        if (row_ok && mine == 0) *reinterpret_cast<uint2*>(out) = make_uint2(0, 0);
        return;
    }
    const float c_exp = in_range(p.scale * kLog2e);
    float ref = kNone, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0 + mine; row_ok && c <= c1; c += BATCH * STEP) {
        float2 ml[BATCH];
        float4 x[BATCH];
        #pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int part = c + k * STEP;
            ml[k] = make_float2(kNone, 0.f);
            x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (part <= c1) {
                // slot 1 of the CTA where the item begins, slot 0 of those where it goes on
                const long long slot = (2LL * part + (part == c0 ? 1 : 0)) * ROWS + r;
                ml[k] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + 2 * slot));
                x[k] = __ldcg(reinterpret_cast<const float4*>(p.part_acc + slot * D + col));
            }
        }
        float top = ref;
        #pragma unroll
        for (int k = 0; k < BATCH; ++k) top = fmaxf(top, ml[k].x);
        const float back = exp2_ftz((ref - top) * c_exp);
        ref = top;
        sum *= back;
        v.x *= back; v.y *= back; v.z *= back; v.w *= back;
        #pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const float f = exp2_ftz((ml[k].x - top) * c_exp);
            sum = fmaf(f, ml[k].y, sum);
            v.x = fmaf(f, x[k].x, v.x); v.y = fmaf(f, x[k].y, v.y); v.z = fmaf(f, x[k].z, v.z); v.w = fmaf(f, x[k].w, v.w);
        }
    }
    if (lane % LPR == 0) sm_ml[group + mine] = make_float2(ref, sum);
    sm_acc[group + mine][lane % LPR] = v;
    __syncthreads();
    if (mine > 0 || !row_ok) return;
    float top = ref;
    #pragma unroll
    for (int k = 1; k < STEP; ++k) top = fmaxf(top, sm_ml[group + k].x);
    sum = 0.f;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
    #pragma unroll
    for (int k = 0; k < STEP; ++k) {
        const float f = exp2_ftz((sm_ml[group + k].x - top) * c_exp);
        const float4 x = sm_acc[group + k][lane % LPR];
        sum = fmaf(f, sm_ml[group + k].y, sum);
        v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
    }
    const float inv = 1.f / sum;
    uint2 o = make_uint2(pack2<BF16>(v.x * inv, v.y * inv), pack2<BF16>(v.z * inv, v.w * inv));
    if (sum == 0.f) o = make_uint2(0, 0);
    *reinterpret_cast<uint2*>(out) = o;
}

}  // namespace bob
