// Host side of the C ABI for rotary positions, the paged cache and the attention over it.
#include "internal.h"
#include "paged.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace bob {

// Return codes as in api.cu.
enum : int { kBadNull = -1, kBadGeom = -2, kBadDtype = -3, kBadHeadDim = -4, kBadStride = -5, kBadWorkspace = -6, kBadDevice = -7,
             kBadLaunch = -8, kBadAttr = -9, kBadAlign = -10 };

// B200's SMs, and not asked of the device: the workspace's size then depends on the arguments alone.
constexpr int kPagedSms = 148;
constexpr int kMaxDevices = 64;

struct CurrentDevice {
    int before = -1;
    bool ok = true, changed = false;
    explicit CurrentDevice(int device) {
        if (device < 0 || device >= kMaxDevices || cudaGetDevice(&before) != cudaSuccess) { ok = false; return; }
        changed = before != device;
        if (changed && cudaSetDevice(device) != cudaSuccess) { ok = false; changed = false; }
    }
    ~CurrentDevice() { if (changed) cudaSetDevice(before); }
};

static int launched() { return cudaGetLastError() == cudaSuccess ? 0 : kBadLaunch; }

static int check_head_dim(int D) { return D == 32 || D == 64 || D == 128 ? 0 : kBadHeadDim; }
static int check_dtype(int dtype) { return dtype == BOB_SM100_FP16 || dtype == BOB_SM100_BF16 ? 0 : kBadDtype; }

// Strides and address of a [B, H, N, D] tensor of tokens; a stride of zero repeats, as of an expanded tensor.
static int check_tokens(const void* ptr, const int64_t* strides) {
    if (!ptr || !strides) return kBadNull;
    if (reinterpret_cast<uintptr_t>(ptr) % 16) return kBadAlign;
    for (int i = 0; i < 3; ++i)
        if (strides[i] < 0 || strides[i] % 8) return kBadStride;
    return 0;
}

static int check_rotary(const bob_sm100_rotary& r, int D) {
    return r.pairs >= 0 && 2 * r.pairs <= D && std::isfinite(r.factor) ? 0 : kBadGeom;
}

static int check_cache(const bob_sm100_cache* c) {
    if (!c) return kBadNull;
    if (int rc = check_dtype(c->dtype)) return rc;
    if (int rc = check_head_dim(c->D)) return rc;
    if (c->pages <= 0 || c->heads <= 0 || c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1))) return kBadGeom;
    if (c->bits != 16 && c->bits != 4) return kBadGeom;
    for (int w = 0; w < 2; ++w) {
        if (!c->data[w] || (c->bits == 4 && !c->scales[w])) return kBadNull;
        if (reinterpret_cast<uintptr_t>(c->data[w]) % 16 || reinterpret_cast<uintptr_t>(c->scales[w]) % 8) return kBadAlign;
        for (int i = 0; i < 3; ++i)
            if (c->strides[w][i] < 0 || c->strides[w][i] % 16 || (c->bits == 4 && (c->scale_strides[w][i] < 0 || c->scale_strides[w][i] % 8))) return kBadStride;
    }
    return 0;
}

static int check_sequences(const bob_sm100_cache* c, const bob_sm100_sequences* s) {
    if (!s || !s->table || !s->lengths) return kBadNull;
    if (s->B <= 0 || s->max_pages <= 0 || s->table_stride < 0 || (int64_t)s->max_pages * c->page_size > (1 << 28)) return kBadGeom;
    return 0;
}

static SequenceParams sequences(const bob_sm100_cache* c, const bob_sm100_sequences* s, bool apart = false) {
    SequenceParams p = {};
    p.table = s->table; p.table_stride = s->table_stride;
    p.lengths = s->lengths; p.counts = s->counts;
    p.B = s->B; p.max_pages = s->max_pages; p.pages = c->pages;
    while ((1 << p.page_shift) < c->page_size) ++p.page_shift;
    p.room = s->max_pages << p.page_shift;
    p.sticky = sticky_word(c->device, true);
    p.first = apart ? -(1 << 29) : 0;
    return p;
}

static CacheTensor cache_tensor(const bob_sm100_cache* c, int w) {
    CacheTensor t = {};
    t.data = static_cast<uint8_t*>(c->data[w]); t.sp = c->strides[w][0]; t.sh = c->strides[w][1]; t.sr = c->strides[w][2];
    t.scales = static_cast<float*>(c->scales[w]);
    t.ssp = c->scale_strides[w][0] / 4; t.ssh = c->scale_strides[w][1] / 4; t.ssr = c->scale_strides[w][2] / 4;
    return t;
}

template <int V> struct Int { static constexpr int value = V; };

template <class F> static void with_form(int form, F f) {
    if (form == kHalf) f(Int<kHalf>{});
    else if (form == kInterleaved) f(Int<kInterleaved>{});
    else if (form == kQuarter) f(Int<kQuarter>{});
    else f(Int<kScattered>{});
}
template <class F> static void with_type(int dtype, F f) {
    if (dtype == BOB_SM100_BF16) f(std::true_type{});
    else f(std::false_type{});
}

// Rows x 16 elements from which on a thread turns four heads and shares its sines between them: with fewer, one each is as
// fast or faster (measured, one head / four, us: 40 rows 2.2 / 2.7, 2,560 rows 2.5 / 3.3, 10,240 rows 3.4 / 3.4, 98,304 rows of 64
// elements 7.1 / 5.4, 163,840 rows 21.1 / 15.4; eight 18.4).
constexpr int64_t kSharedTurns = (int64_t)kPagedSms * 512;

static int run_rotate(const bob_sm100_rotate_args* a, cudaStream_t stream, const int* lengths = nullptr, const int* counts = nullptr, int pack = 1) {
    RotateParams p = {};
    p.lengths = lengths; p.counts = counts; p.pack = pack;
    p.rotary = a->rotary;
    if (a->inverse)
        for (uint64_t& x : p.rotary.turns) x = 0 - x;
    for (int i = 0; i < 2; ++i) {
        p.t[i].in = static_cast<const uint16_t*>(a->in[i]);
        p.t[i].in_sb = a->in_strides[i][0]; p.t[i].in_sh = a->in_strides[i][1]; p.t[i].in_sn = a->in_strides[i][2];
        p.t[i].out = static_cast<uint16_t*>(a->out[i]);
        p.t[i].H = a->heads[i];
    }
    p.B = a->B; p.N = a->N; p.D = a->D;
    p.positions = a->positions; p.wide = a->position_bits == 64;
    p.pos_sb = a->position_strides[0]; p.pos_sn = a->position_strides[1];
    p.first = a->first;
    const int64_t threads = (int64_t)a->B * a->N * (a->D / 16), blocks = (threads + kRotateThreads - 1) / kRotateThreads;
    const int heads = a->heads[0] + a->heads[1];
    if (blocks > 0x7fffffffLL) return kBadGeom;
    with_form(rotary_form(&a->rotary), [&](auto form) {
        with_type(a->dtype, [&](auto bf16) {
            constexpr int F = decltype(form)::value;
            constexpr bool BF = decltype(bf16)::value;
            auto go = [&](auto hpt) {
                constexpr int HPT = decltype(hpt)::value;
                const dim3 grid((unsigned)blocks, (heads + HPT - 1) / HPT);
                rotate_kernel<F, BF, HPT><<<grid, kRotateThreads, 0, stream>>>(p);
            };
            if (threads * heads >= kSharedTurns) go(Int<4>{});
            else go(Int<1>{});
        });
    });
    return launched();
}

static int run_append(const bob_sm100_cache* c, const bob_sm100_sequences* s, const bob_sm100_rotary* r, int N, const void* const* in,
                      const int64_t* const* strides, cudaStream_t stream) {
    AppendParams p = {};
    p.rotary = *r;
    p.seq = sequences(c, s);
    for (int w = 0; w < 2; ++w) {
        p.cache[w] = cache_tensor(c, w);
        p.in[w] = static_cast<const uint16_t*>(in[w]);
        p.in_sb[w] = strides[w][0]; p.in_sh[w] = strides[w][1]; p.in_sn[w] = strides[w][2];
    }
    p.H = c->heads; p.N = N; p.D = c->D;
    const int64_t threads = (int64_t)s->B * N * (c->D / 16);
    // 4 bits: several heads to a thread, which share its 64-bit sines, where enough threads are left (measured, one / two / four /
    // eight heads, us: 512 rows of 128 elements 4.6 / 5.8 / 8.4 / 13.4, 96,000 rows 42.7 / 34.2 / 31.3 / 31.0, 128,032 rows of 64
    // 28.0 / 23.3 / 21.6 / 19.8).  16 bits: one (98 MB 19.5; with two 19.1, four 20.5).
    p.heads_each = 1;
    if (c->bits == 4)
        while (p.heads_each < 8 && threads * c->heads / (2 * p.heads_each) >= kPagedSms * 384) p.heads_each *= 2;
    const int64_t blocks = (threads + kCacheThreads - 1) / kCacheThreads;
    if (blocks > 0x7fffffffLL) return kBadGeom;
    with_form(rotary_form(r), [&](auto form) {
        with_type(c->dtype, [&](auto bf16) {
            constexpr int F = decltype(form)::value;
            constexpr bool BF = decltype(bf16)::value;
            const dim3 grid((unsigned)blocks, (c->heads + p.heads_each - 1) / p.heads_each);
            if (c->bits == 16) append_kernel<F, BF, 16><<<grid, kCacheThreads, 0, stream>>>(p);
            else append_kernel<F, BF, 4><<<grid, kCacheThreads, 0, stream>>>(p);
        });
    });
    return launched();
}

// unpack > 0: for a paged call of that many rows per sequence (ReadParams::unpack).
static int run_read(const bob_sm100_cache* c, const bob_sm100_sequences* s, int n, void* const* out, cudaStream_t stream, bool apart = false, int unpack = 0, int window = 0, int out_pages = 0, int out_shift = 0) {
    ReadParams p = {};
    p.seq = sequences(c, s, apart);
    if (!unpack) p.seq.counts = nullptr;
    p.unpack = unpack;
    p.window = window;
    p.out_pages = out_pages; p.out_shift = out_shift;
    for (int w = 0; w < 2; ++w) { p.cache[w] = cache_tensor(c, w); p.out[w] = static_cast<uint16_t*>(out[w]); }
    p.H = c->heads; p.N = n; p.D = c->D;
    int64_t blocks = ((int64_t)s->B * n * (c->D / 16) + kCacheThreads - 1) / kCacheThreads;
    if (unpack) {                                        // as many CTAs as run at once, or whole sequences' worth
        const int64_t most = ((int64_t)n * (c->D / 16) + kCacheThreads - 1) / kCacheThreads;
        p.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(most, kPagedSms * 2048 / kCacheThreads / ((int64_t)s->B * c->heads)));
        blocks = (int64_t)p.chunks * s->B;
    }
    if (blocks > 0x7fffffffLL) return kBadGeom;
    with_type(c->dtype, [&](auto bf16) {
        constexpr bool BF = decltype(bf16)::value;
        const dim3 grid((unsigned)blocks, c->heads);
        auto run = [&](auto kernel) { kernel<<<grid, kCacheThreads, 0, stream>>>(p); };
        if (c->bits == 16) run(unpack ? read_kernel<BF, 16, true> : read_kernel<BF, 16, false>);
        else run(unpack ? read_kernel<BF, 4, true> : read_kernel<BF, 4, false>);
    });
    return launched();
}

// ---- attention --------------------------------------------------------------------------------------------------
static size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// sweep: through the kernel for many rows, after a kernel that turns the queries into the workspace (and, in 4 bits, one that
// unpacks the cache there, or brings it into larger pages: kv_bytes > 0), and with splits > 1 before one that adds the parts.
struct PagedPlan { bool sweep; int pack, splits, rows, groups, ctas; int out_pages, out_shift; size_t q_offset, ml_offset, acc_offset, kv_offset, kv_bytes, bytes; };

// Most rows of a KV head's queries that paged_kernel takes: 32 in 16 bits (16 but for fewer than 4 heads in all), 64 in 4 bits.
// Measured, paged_kernel / tiles of 128 rows, us: 20 rows of 8 heads in 16 bits 300 keys 20.0 / 20.8, 3000 25.2 / 22.7, of 64
// heads 25.1 / 20.5 and 49.8 / 37.4; 32 rows of one head 14.2 / 20.9 and 15.9 / 21.0.  In 4 bits unpacking costs what tiles
// gain, us: 8 sequences x 64 heads x 20 rows, 1000 keys 121 / 147 (fp16, in which rows are taken 16 at a time, 128 / 147), one sequence of
// 8 heads, 8192 keys 43 / 35 (30 / 35); 4 sequences x 8 heads x 64 rows, 4096 keys 45 / 50 (56 / 49); 3 sequences x 16 heads x 100
// rows, 2500 keys 87 / 50 (83 / 51), 500 49 / 28.
constexpr int kPagedRows = 32, kPagedRows4 = 64;
// ... while the unpacked cache (as much as the page table has room for) takes no more than this.
constexpr int64_t kMostUnpacked = (int64_t)1 << 30;
// Tiles of a KV head from which on 16-bit pages of 16 rows, whose copies of 2 KB hold a tile up, are brought into larger ones first (of up
// to 8192 keys in pages of 16, as they are / in larger pages, us: 4 tiles 138 / 142, 8 tiles 257 / 222, 32 tiles 793 / 590; pages of 32 rows
// 198 / 216 and 597 / 594).
constexpr int kRepagedTiles = 8;
constexpr int kMostSplits = 16;
// Query heads that may share a KV head (PagedParams::g_part).
constexpr int kMostGroup = 32;

static int block_keys(int D, int bits) { return bits == 16 ? 2048 / D : (D == 128 ? 32 : 64); }

// The kernel for many rows takes its queries as tiles of 128 rows of a head: those to be turned, and expanded ones, are written
// out first, and so are those of heads that share keys where that makes at most half as many tiles.
static int packed_heads(const bob_sm100_paged_args* a) {
    const int64_t G = a->Hq / a->cache.heads, apart = (a->N + 127) / 128 * G, together = (a->N * G + 127) / 128;
    return 2 * together <= apart ? (int)G : 1;
}
static bool copies_queries(const bob_sm100_paged_args* a) {
    const int64_t* s = a->q_strides;
    return a->rotary.pairs || packed_heads(a) > 1 || (s[0] == 0 && a->seq.B > 1) || (s[1] == 0 && a->Hq > 1) || (s[2] == 0 && a->N > 1);
}

static PagedPlan paged_plan(const bob_sm100_paged_args* a) {
    PagedPlan d = {};
    const int64_t R = (int64_t)a->N * (a->Hq / a->cache.heads);
    const int64_t rows = (int64_t)a->seq.B * a->Hq * a->N;
    // the cache unpacked, in pages of a tile's 128 rows or more
    for (d.out_shift = 7; (1 << d.out_shift) < a->cache.page_size;) ++d.out_shift;
    d.out_pages = (int)(((int64_t)a->seq.max_pages * a->cache.page_size + (1 << d.out_shift) - 1) >> d.out_shift);
    const int64_t unpacked = ((int64_t)a->seq.B * d.out_pages << d.out_shift) * a->cache.heads * a->cache.D * 2;
    d.sweep = a->cache.bits == 16 ? R > kPagedRows || (R > 16 && (int64_t)a->seq.B * a->cache.heads >= 4) : R > kPagedRows4 && 2 * unpacked <= kMostUnpacked;
    if (d.sweep) {
        // with a tile for fewer than half of the SMs, the keys are divided too (whatever the lengths are)
        d.pack = packed_heads(a);
        const int64_t items = ((int64_t)a->N * d.pack + 127) / 128 * (a->Hq / d.pack) * a->seq.B;
        d.splits = (int)std::max<int64_t>(1, std::min<int64_t>(kMostSplits, kPagedSms / items));
        const bool parted = d.splits > 1 || d.pack > 1;
        d.q_offset = 256;
        d.ml_offset = d.q_offset + (copies_queries(a) ? up256(rows * a->cache.D * 2) : 0);
        d.acc_offset = d.ml_offset + (parted ? up256(d.splits * rows * 2 * sizeof(float)) : 0);
        d.kv_offset = d.acc_offset + (parted ? up256(d.splits * rows * a->cache.D * sizeof(float)) : 0);
        const int64_t tiles = ((int64_t)a->N * d.pack + 127) / 128 * (a->Hq / a->cache.heads / d.pack);       // of a KV head
        const bool repaged = a->cache.page_size == 16 && tiles >= kRepagedTiles && 2 * unpacked <= kMostUnpacked;
        d.kv_bytes = a->cache.bits == 4 || repaged ? up256(unpacked) : 0;
        d.bytes = d.kv_offset + 2 * d.kv_bytes;
        return d;
    }
    // fp16 over 4 bits: 16 at a time, since one part of a probability times its scale is a bf16 number, which has 3 bits fewer
    // than the rest of the call (error against 64 bits 1.8e-3 with 32 rows at a time, 2.1e-4 with 16; us, 32 / 16 at a time: 8 sequences x
    // 64 heads x 20 rows of 64 elements, 1000 keys 56 / 75, 8192 keys 217 / 338; 4 x 8 heads x 64 rows, 4096 keys 26 / 33; 8 x 8 heads x 20
    // rows of 128 elements, 3000 keys 55 / 48)
    const bool by16 = a->cache.bits == 4 && a->cache.dtype == BOB_SM100_FP16;
    d.rows = R <= 8 ? 8 : (R <= 16 || by16 ? 16 : 32);
    d.groups = (int)((R + d.rows - 1) / d.rows);
    // no more CTAs than the longest possible sequences have work for
    const int64_t kb = block_keys(a->cache.D, a->cache.bits), most = ((int64_t)a->seq.max_pages * a->cache.page_size + kb - 1) / kb;
    const int64_t line = most * a->seq.B * a->cache.heads * d.groups;
    d.ctas = (int)std::min<int64_t>((d.rows == 8 ? 3 : 2) * kPagedSms, std::max<int64_t>(1, line / kPagedMinBlocks));
    const size_t slots = (size_t)d.ctas * 2 * d.rows;
    d.acc_offset = up256(slots * 2 * sizeof(float));
    d.bytes = d.acc_offset + slots * a->cache.D * sizeof(float);
    return d;
}

static int check_paged(const bob_sm100_paged_args* a) {
    if (!a) return kBadNull;
    if (int rc = check_cache(&a->cache)) return rc;
    if (int rc = check_sequences(&a->cache, &a->seq)) return rc;
    if (int rc = check_rotary(a->rotary, a->cache.D)) return rc;
    if (a->Hq <= 0 || a->Hq % a->cache.heads || a->N <= 0 || a->N > (1 << 28)) return kBadGeom;
    if (a->Hq / a->cache.heads > kMostGroup) return kBadGeom;
    if (a->window < 0 || (a->window > 0 && !a->is_causal)) return kBadGeom;
    if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return kBadGeom;
    if (int rc = check_tokens(a->q, a->q_strides)) return rc;
    if (!a->out) return kBadNull;
    if (reinterpret_cast<uintptr_t>(a->out) % 16) return kBadAlign;
    if ((int64_t)a->N * (a->Hq / a->cache.heads) > (1 << 28)) return kBadGeom;
    const PagedPlan d = paged_plan(a);
    if (!d.sweep) {
        // a sequence's part of the line, and the grid of the second kernel, are counted in 32 bits
        const int64_t kb = block_keys(a->cache.D, a->cache.bits), blocks = ((int64_t)a->seq.max_pages * a->cache.page_size + kb - 1) / kb;
        if (blocks * a->cache.heads * d.groups > 0x7fffffffLL || (int64_t)a->seq.B * a->cache.heads * d.groups > 0x7fffffffLL) return kBadGeom;
    }
    return 0;
}

template <int D, int ROWS, bool BF16, int BITS>
static int launch_paged(PagedParams& p, int device, cudaStream_t stream) {
    using CFG = PagedConfig<D, ROWS, BITS>;
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = 1ull << device;
    if (!(done.load(std::memory_order_acquire) & bit)) {
        if (cudaFuncSetAttribute(paged_kernel<D, ROWS, BF16, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, CFG::SMEM) != cudaSuccess) return kBadAttr;
        done.fetch_or(bit, std::memory_order_release);
    }
    paged_kernel<D, ROWS, BF16, BITS><<<p.ctas, kPagedThreads, CFG::SMEM, stream>>>(p);
    if (int rc = launched()) return rc;
    // started while paged_kernel runs, and waits for it
    cudaLaunchAttribute early = {};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    const int64_t items = (int64_t)p.seq.B * p.Hkv * p.groups;
    const int rows = std::min(ROWS, p.N * p.G);
    cfg.blockDim = dim3(kPagedThreads);
    cfg.stream = stream;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    // a CTA to a row while all of them run at once (the whole call, a warp / four to a row,
    // us: 512 rows in 9 parts each 29.3 / 28.8, 128 rows in 74 parts 31.1 / 30.2)
    if (items * rows <= kPagedSms * 8) {
        cfg.gridDim = dim3((unsigned)items, (unsigned)rows);
        return cudaLaunchKernelEx(&cfg, combine_kernel<D, ROWS, BF16, BITS, 4>, p) == cudaSuccess ? 0 : kBadLaunch;
    }
    cfg.gridDim = dim3((unsigned)items, (unsigned)((rows + kPagedWarps - 1) / kPagedWarps));
    return cudaLaunchKernelEx(&cfg, combine_kernel<D, ROWS, BF16, BITS, 1>, p) == cudaSuccess ? 0 : kBadLaunch;
}

static int run_paged(const bob_sm100_paged_args* a, void* workspace, cudaStream_t stream) {
    const PagedPlan d = paged_plan(a);
    if (d.sweep) {
        char* ws = static_cast<char*>(workspace);
        bob_sm100_paged_args b = *a;
        SequenceParams seq = sequences(&a->cache, &a->seq, !a->is_causal);
        const void* q = a->q;
        int64_t strides[3] = {a->q_strides[0], a->q_strides[1], a->q_strides[2]};
        if (copies_queries(a)) {
            bob_sm100_rotate_args r = {};
            r.B = a->seq.B; r.N = a->N; r.D = a->cache.D; r.dtype = a->cache.dtype; r.device = a->cache.device;
            r.heads[0] = a->Hq;
            r.in[0] = q;
            for (int i = 0; i < 3; ++i) r.in_strides[0][i] = strides[i];
            r.out[0] = ws + d.q_offset;
            r.rotary = a->rotary;
            if (int rc = run_rotate(&r, stream, a->seq.lengths, a->seq.counts, d.pack)) return rc;
            q = r.out[0];
            strides[2] = a->cache.D; strides[1] = strides[2] * a->N * d.pack; strides[0] = strides[1] * (a->Hq / d.pack);
        }
        if (d.kv_bytes) {
            bob_sm100_cache& c = b.cache;
            c.page_size = 1 << d.out_shift;
            for (int w = 0; w < 2; ++w) {
                c.data[w] = ws + d.kv_offset + w * d.kv_bytes;
                c.strides[w][2] = 2 * c.D; c.strides[w][1] = c.strides[w][2] * c.page_size; c.strides[w][0] = c.strides[w][1] * c.heads;
            }
            if (int rc = run_read(&a->cache, &a->seq, seq.room, c.data, stream, !a->is_causal, a->N, std::min(a->window, 1 << 28), d.out_pages, d.out_shift)) return rc;
            c.bits = 16;
            seq.max_pages = d.out_pages; seq.page_shift = d.out_shift;
            c.pages = seq.pages = seq.B * seq.max_pages;
            seq.table = nullptr;
        }
        float* ml = reinterpret_cast<float*>(ws + d.ml_offset);
        float* acc = reinterpret_cast<float*>(ws + d.acc_offset);
        if (int rc = sweep_paged(&b, seq, q, strides, d.pack, d.splits, acc, ml, workspace, stream)) return rc;
        if (d.splits == 1 && d.pack == 1) return 0;
        const int64_t rows = (int64_t)a->seq.B * a->Hq * a->N, blocks = (rows * (a->cache.D / 4) + 255) / 256;
        with_type(a->cache.dtype, [&](auto bf16) {
            add_splits_kernel<decltype(bf16)::value><<<(unsigned)blocks, 256, 0, stream>>>(ml, acc, static_cast<uint16_t*>(a->out), d.splits, rows, a->cache.D, a->N, d.pack, a->scale);
        });
        return launched();
    }
    PagedParams p = {};
    p.rotary = a->rotary;
    p.seq = sequences(&a->cache, &a->seq, !a->is_causal);
    for (int w = 0; w < 2; ++w) p.cache[w] = cache_tensor(&a->cache, w);
    p.q = static_cast<const uint16_t*>(a->q); p.q_sb = a->q_strides[0]; p.q_sh = a->q_strides[1]; p.q_sn = a->q_strides[2];
    p.out = static_cast<uint16_t*>(a->out);
    p.Hq = a->Hq; p.Hkv = a->cache.heads; p.G = a->Hq / a->cache.heads; p.N = a->N;
    p.g_part = 65536 / p.G + 1;
    p.form = rotary_form(&a->rotary);
    p.groups = d.groups;
    p.causal = a->is_causal != 0;
    p.window = std::min(a->window, 1 << 28);
    p.scale = a->scale;
    p.ctas = d.ctas;
    auto same = [](const int64_t (&x)[2][3]) { return std::equal(x[0], x[0] + 3, x[1]); };
    p.alike = same(a->cache.strides) && (a->cache.bits == 16 || same(a->cache.scale_strides));
    p.part_ml = static_cast<float*>(workspace);
    p.part_acc = reinterpret_cast<float*>(static_cast<char*>(workspace) + d.acc_offset);
    int rc = 0;
    with_type(a->cache.dtype, [&](auto bf16) {
        constexpr bool BF = decltype(bf16)::value;
        auto dim = [&](auto rows, auto bits) {
            constexpr int ROWS = decltype(rows)::value, BITS = decltype(bits)::value;
            if constexpr (ROWS == 32 && BITS == 4 && !BF) rc = kBadGeom;      // (paged_plan takes 16 at a time)
            else if (a->cache.D == 32) rc = launch_paged<32, ROWS, BF, BITS>(p, a->cache.device, stream);
            else if (a->cache.D == 64) rc = launch_paged<64, ROWS, BF, BITS>(p, a->cache.device, stream);
            else rc = launch_paged<128, ROWS, BF, BITS>(p, a->cache.device, stream);
        };
        auto width = [&](auto bits) {
            if (d.rows == 8) dim(Int<8>{}, bits);
            else if (d.rows == 16) dim(Int<16>{}, bits);
            else dim(Int<32>{}, bits);
        };
        if (a->cache.bits == 16) width(Int<16>{}); else width(Int<4>{});
    });
    return rc;
}

}  // namespace bob

using namespace bob;

extern "C" int bob_sm100_rotate(const bob_sm100_rotate_args* a, void* stream) {
    if (!a) return kBadNull;
    if (int rc = check_dtype(a->dtype)) return rc;
    if (int rc = check_head_dim(a->D)) return rc;
    if (int rc = check_rotary(a->rotary, a->D)) return rc;
    if (a->B <= 0 || a->N <= 0 || a->N > (1 << 28) || a->heads[0] <= 0 || a->heads[1] < 0 || (int64_t)a->heads[0] + a->heads[1] > 65535) return kBadGeom;
    if (a->positions && a->position_bits != 32 && a->position_bits != 64) return kBadGeom;
    for (int i = 0; i < (a->heads[1] ? 2 : 1); ++i) {
        if (int rc = check_tokens(a->in[i], a->in_strides[i])) return rc;
        if (!a->out[i]) return kBadNull;
        if (reinterpret_cast<uintptr_t>(a->out[i]) % 16) return kBadAlign;
    }
    CurrentDevice device(a->device);
    if (!device.ok) return kBadDevice;
    return run_rotate(a, static_cast<cudaStream_t>(stream));
}

extern "C" int bob_sm100_cache_append(const bob_sm100_cache* c, const bob_sm100_sequences* s, const bob_sm100_rotary* r, int N,
                                      const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, void* stream) {
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_sequences(c, s)) return rc;
    if (!r) return kBadNull;
    if (int rc = check_rotary(*r, c->D)) return rc;
    if (N <= 0 || N > (1 << 28) || c->heads > 65535) return kBadGeom;
    if (int rc = check_tokens(k, k_strides)) return rc;
    if (int rc = check_tokens(v, v_strides)) return rc;
    CurrentDevice device(c->device);
    if (!device.ok) return kBadDevice;
    const void* in[2] = {k, v};
    const int64_t* strides[2] = {k_strides, v_strides};
    return run_append(c, s, r, N, in, strides, static_cast<cudaStream_t>(stream));
}

extern "C" int bob_sm100_cache_read(const bob_sm100_cache* c, const bob_sm100_sequences* s, int n, void* k, void* v, void* stream) {
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_sequences(c, s)) return rc;
    if (n <= 0 || n > (1 << 28) || c->heads > 65535) return kBadGeom;
    if (!k || !v) return kBadNull;
    if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16) return kBadAlign;
    CurrentDevice device(c->device);
    if (!device.ok) return kBadDevice;
    void* out[2] = {k, v};
    return run_read(c, s, n, out, static_cast<cudaStream_t>(stream));
}

extern "C" size_t bob_sm100_paged_workspace_bytes(const bob_sm100_paged_args* a) {
    return check_paged(a) ? 0 : paged_plan(a).bytes;
}

extern "C" int bob_sm100_paged_fwd(const bob_sm100_paged_args* a, void* workspace, void* stream) {
    if (int rc = check_paged(a)) return rc;
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256) return kBadWorkspace;
    CurrentDevice device(a->cache.device);
    if (!device.ok) return kBadDevice;
    return run_paged(a, workspace, static_cast<cudaStream_t>(stream));
}
