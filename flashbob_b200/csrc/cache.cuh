// The paged cache of keys and values: new rows into its pages, and pages back into contiguous rows.
//
// A page holds page_size positions of every KV head.  Position t of sequence b lies in page page_table[b][t / page_size],
// row t % page_size.  lengths[b] counts the positions that are there with the new ones, counts[b] the new ones, so new
// row i sits at position lengths[b] - counts[b] + i, as a query of the same call does.
//
// In 4 bits a row of a head (D elements) is kept as codes 0 ... 15, element 2 j in the low half of byte j, and fp32
// (scale, zero): value = code * scale + zero, zero = the row's minimum, scale = (maximum - minimum) times the fp32 number
// 1/15, or 1 where they are equal; code = (element - zero) / scale to the nearest, halves to even.  A row with a NaN or an infinity reads as NaN or infinities.
//
// What bounds these kernels: every row is read and written once.  Page entries and lengths are checked here, for they are
// known on the GPU only: an entry outside the cache is reported and its rows are neither read nor written.
//
// Measured (replayed in a graph): ragged prompts up to 2048 tokens, 8 x 8 heads of 128 elements in 16 bits 20.8 us (92 MB, 4.4 TB/s; 27.3 for
// 134 MB without raggedness), read back 20.2 (113 MB, 5.6 TB/s); up to 4001 tokens, 2 x 16 heads of 64 elements into 4 bits 19.0 us (the
// exact rotation and the quotients: instructions), read back 10.3; one token of 64 sequences x 8 heads of 128 elements 2.8, 4 bits 4.7.
#pragma once

#include "rotary.cuh"
#include "sequence.cuh"

namespace bob {

struct CacheTensor {
    uint8_t* data; long long sp, sh, sr;                         // byte strides: page, head, row
    float* scales; long long ssp, ssh, ssr;                      // 4 bits: (scale, zero) of a row; strides in floats
};

struct alignas(16) AppendParams {
    bob_sm100_rotary rotary;
    SequenceParams seq;
    CacheTensor cache[2];                                        // keys, values
    const uint16_t* in[2]; long long in_sb[2], in_sh[2], in_sn[2];
    int H, N, D, heads_each;
};

struct ReadParams {
    SequenceParams seq;
    CacheTensor cache[2];
    uint16_t* out[2];                                            // contiguous [B, H, N, D]
    int H, N, D;
    // unpacking: out is [B * out_pages, H, 1 << out_shift, D], page i of sequence b at b * out_pages + i, and only rows that a paged
    // call of `unpack` rows per sequence looks at are written
    int unpack, window, out_pages, out_shift, chunks;
};

__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// Quantises a row of D = 16 * per_row elements, 16 of them in each of per_row neighbouring lanes (all lanes of the warp
// call this).  Every operation is rounded to nearest in fp32, so the codes are those of the formula in plain arithmetic.  The
// quotient is Markstein's: with y the rounded reciprocal of b, q = a y and r = a - b q (one rounding, exact), q + r y is
// a / b correctly rounded.  (Rows of 8-bit mantissas have quotients on the border between two codes all the time, so an
// approximate quotient with a division for those near a border costs more: 65 us on 63 MB against 44 without.)
template <bool BF16>
__device__ __forceinline__ uint2 quantise16(const Chunks& x, int per_row, float& scale, float& zero) {
    float v[16];
    widen8<BF16>(x.a, v);
    widen8<BF16>(x.b, v + 8);
    float lo = v[0], hi = v[0];
    #pragma unroll
    for (int i = 1; i < 16; ++i) { lo = min_nan(lo, v[i]); hi = max_nan(hi, v[i]); }
    for (int o = 1; o < per_row; o <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    zero = lo;
    scale = hi > lo ? __fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f) : 1.f;
    const float inv = __frcp_rn(scale);
    // q + 1.5 * 2^23 rounds q to a whole number, halves to even, in the last bits: its bits are kWhole + code, and eight of
    // them, each 16 times the one before, add up to the word of codes and a constant
    constexpr float kShift = 12582912.f;
    constexpr uint32_t kWhole = 0x4b400000u, kExtra = kWhole * 0x11111111u;
    uint32_t word[2] = {0, 0};
    if (scale > 1e-30f && scale < 1e30f) {                       // nothing here overflows or gets too small to be exact
        #pragma unroll
        for (int i = 15; i >= 0; --i) {
            const float d = __fsub_rn(v[i], lo), q = __fmul_rn(d, inv);
            word[i >> 3] = word[i >> 3] * 16 + __float_as_uint(__fadd_rn(__fmaf_rn(__fmaf_rn(-q, scale, d), inv, q), kShift));
        }
    } else {
        const uint32_t w[8] = {x.a.x, x.a.y, x.a.z, x.a.w, x.b.x, x.b.y, x.b.z, x.b.w};
        #pragma unroll 1
        for (int i = 15; i >= 0; --i) {
            uint32_t pair = w[0];
            #pragma unroll
            for (int j = 1; j < 8; ++j) pair = i / 2 == j ? w[j] : pair;
            const uint16_t bits = static_cast<uint16_t>(i % 2 ? pair >> 16 : pair);
            const float e = BF16 ? __uint_as_float(static_cast<uint32_t>(bits) << 16) : __half2float(__ushort_as_half(bits));
            const uint32_t r = __float_as_uint(__fadd_rn(__fdiv_rn(__fsub_rn(e, lo), scale), kShift));
            if (i < 8) word[0] = word[0] * 16 + r; else word[1] = word[1] * 16 + r;
        }
    }
    return make_uint2(word[0] - kExtra, word[1] - kExtra);
}

constexpr int kCacheThreads = 256;

// One thread: 16 elements of a new row, of one head (blockIdx.y) or, with the same sines, of several: keys and values.  BITS 4 turns the keys in 64 bits: a
// rounding that falls the other way can move an element by a whole step of the 4-bit row, 1/15 of its range.
template <int FORM, bool BF16, int BITS>
__global__ void __launch_bounds__(kCacheThreads) append_kernel(const __grid_constant__ AppendParams p) {
    __shared__ __align__(16) uint16_t stage[FORM == kScattered ? kCacheThreads * 16 : 8];
    const int each = BITS == 4 ? p.heads_each : 1, per_row = p.D / 16, h0 = blockIdx.y * each, h1 = min(p.H, h0 + each);
    const long long id = (long long)blockIdx.x * kCacheThreads + threadIdx.x, token = id / per_row;
    const int c = static_cast<int>(id % per_row);
    const int b = token < (long long)p.seq.B * p.N ? static_cast<int>(token / p.N) : -1, n = static_cast<int>(token % p.N);
    // the lanes of a row agree on everything here; those without a row stay for the shuffles
    bool there = b >= 0;
    int page = 0, position = 0;
    if (there) {
        const Sequence s = sequence_of(p.seq, b, p.N);
        if (n == 0 && c == 0 && h0 == 0 && !s.ok) report(p.seq.sticky, kStatusBadLength);
        position = s.start + n;
        there = n < s.count;
        if (there) {
            page = page_of(p.seq, b, position);
            if (page < 0) { report(p.seq.sticky, kStatusBadPage); there = false; }
        }
    }
    if (__ballot_sync(0xffffffffu, there) == 0) return;
    const int row = position & ((1 << p.seq.page_shift) - 1);
    const RowPlace<FORM> place(c, p.rotary.pairs);
    const RowPlace<kInterleaved> plain(c, 0);                    // 16 elements in a row
    const auto outer = outer_place(place, plain);
    const uint16_t* src_k = p.in[0] + b * p.in_sb[0] + n * p.in_sn[0];
    const uint16_t* src_v = p.in[1] + b * p.in_sb[1] + n * p.in_sn[1];
    uint8_t* const page_k = p.cache[0].data + page * p.cache[0].sp + row * p.cache[0].sr;
    uint8_t* const page_v = p.cache[1].data + page * p.cache[1].sp + row * p.cache[1].sr;
    auto fetch = [&](int h, Chunks& k, Chunks& v) {
        k = v = Chunks{};
        if (!there) return;
        k = outer.load(src_k + h * p.in_sh[0]);
        v = plain.load(src_v + h * p.in_sh[1]);
    };
    Chunks next_k, next_v;
    fetch(h0, next_k, next_v);
    Turner<FORM, BF16, std::conditional_t<BITS == 4, double, float>> turn;
    turn.set(p.rotary, c, position);
    #pragma unroll 1
    for (int h = h0; h < h1; ++h) {
        const Chunks k = turned<FORM>(turn, place, plain, next_k, stage + threadIdx.x / per_row * p.D), v = next_v;
        if (h + 1 < h1) fetch(h + 1, next_k, next_v);
        uint8_t* const dst_k = page_k + h * p.cache[0].sh;
        uint8_t* const dst_v = page_v + h * p.cache[1].sh;
        if constexpr (BITS == 16) {
            if (!there) continue;
            outer.store(reinterpret_cast<uint16_t*>(dst_k), k);
            plain.store(reinterpret_cast<uint16_t*>(dst_v), v);
        } else {
            float2 sk, sv;
            const uint2 ck = quantise16<BF16>(k, per_row, sk.x, sk.y), cv = quantise16<BF16>(v, per_row, sv.x, sv.y);
            if (!there) continue;
            if constexpr (FORM == kQuarter) {
                *reinterpret_cast<uint16_t*>(dst_k + place.element(0, false) / 2) = static_cast<uint16_t>(ck.x);
                *reinterpret_cast<uint16_t*>(dst_k + place.element(4, false) / 2) = static_cast<uint16_t>(ck.x >> 16);
                *reinterpret_cast<uint16_t*>(dst_k + place.element(0, true) / 2) = static_cast<uint16_t>(ck.y);
                *reinterpret_cast<uint16_t*>(dst_k + place.element(4, true) / 2) = static_cast<uint16_t>(ck.y >> 16);
            } else {
                *reinterpret_cast<uint32_t*>(dst_k + outer.first / 2) = ck.x;
                *reinterpret_cast<uint32_t*>(dst_k + outer.second / 2) = ck.y;
            }
            *reinterpret_cast<uint2*>(dst_v + 8 * c) = cv;
            if (c == 0) {
                *reinterpret_cast<float2*>(p.cache[0].scales + page * p.cache[0].ssp + h * p.cache[0].ssh + row * p.cache[0].ssr) = sk;
                *reinterpret_cast<float2*>(p.cache[1].scales + page * p.cache[1].ssp + h * p.cache[1].ssh + row * p.cache[1].ssr) = sv;
            }
        }
    }
}

// 16 elements of row n of sequence b and head h.
template <bool BF16, int BITS, bool UNPACK>
__device__ __forceinline__ void read_piece(const ReadParams& p, const Sequence& s, int b, int h, int n, int c) {
    int page = -1;
    if (n < s.length) {
        page = page_of(p.seq, b, n);
        if (page < 0) report(p.seq.sticky, kStatusBadPage);
    }
    const int row = n & ((1 << p.seq.page_shift) - 1);
    Chunks x[2];
    uint2 code[2] = {};
    float2 sc[2] = {};
    #pragma unroll
    for (int w = 0; w < 2; ++w) {
        x[w] = Chunks{};
        if (page < 0) continue;
        const CacheTensor& t = p.cache[w];
        const uint8_t* src = t.data + page * t.sp + h * t.sh + row * t.sr;
        if constexpr (BITS == 16) {
            x[w].a = __ldg(reinterpret_cast<const uint4*>(src) + 2 * c);
            x[w].b = __ldg(reinterpret_cast<const uint4*>(src) + 2 * c + 1);
        } else {
            code[w] = __ldg(reinterpret_cast<const uint2*>(src) + c);
            sc[w] = __ldg(reinterpret_cast<const float2*>(t.scales + page * t.ssp + h * t.ssh + row * t.ssr));
        }
    }
    #pragma unroll
    for (int w = 0; w < 2; ++w) {
        if constexpr (BITS == 4) {
            float v[16];
            #pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = fmaf(static_cast<float>(((j < 8 ? code[w].x : code[w].y) >> (4 * (j & 7))) & 15u), sc[w].x, sc[w].y);
            x[w].a = narrow8<BF16>(v);
            x[w].b = narrow8<BF16>(v + 8);
        }
        const long long at = UNPACK ? (((long long)b * p.out_pages + (n >> p.out_shift)) * p.H + h << p.out_shift) + (n & ((1 << p.out_shift) - 1))
                                      : ((long long)b * p.H + h) * p.N + n;
        uint4* dst = reinterpret_cast<uint4*>(p.out[w] + at * p.D) + 2 * c;
        dst[0] = x[w].a;
        dst[1] = x[w].b;
    }
}

// One thread: 16 elements of a cached row of a head (blockIdx.y), of keys and values.  Rows behind a sequence become zero.
// Unpacking, `chunks` CTAs to a sequence take its rows in turn: a page table has room for more than a sequence holds.
template <bool BF16, int BITS, bool UNPACK>
__global__ void __launch_bounds__(kCacheThreads) read_kernel(const __grid_constant__ ReadParams p) {
    const int per_row = p.D / 16, h = blockIdx.y;
    if constexpr (UNPACK) {
        const int b = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks, c = threadIdx.x % per_row;
        const Sequence s = sequence_of(p.seq, b, p.unpack);
        if (blockIdx.x % p.chunks == 0 && threadIdx.x == 0 && h == 0 && !s.ok) report(p.seq.sticky, kStatusBadLength);
        const int first = p.window > 0 ? max(0, s.start - p.window + 1) : 0;
        for (long long n = first + (chunk * kCacheThreads + threadIdx.x) / per_row; n < s.length; n += p.chunks * (kCacheThreads / per_row))
            read_piece<BF16, BITS, UNPACK>(p, s, b, h, static_cast<int>(n), c);
        return;
    }
    const long long id = (long long)blockIdx.x * kCacheThreads + threadIdx.x, token = id / per_row;
    if (token >= (long long)p.seq.B * p.N) return;
    const int c = static_cast<int>(id % per_row), b = static_cast<int>(token / p.N), n = static_cast<int>(token % p.N);
    const Sequence s = sequence_of(p.seq, b, 0);
    if (n == 0 && c == 0 && h == 0 && !s.ok) report(p.seq.sticky, kStatusBadLength);
    read_piece<BF16, BITS, UNPACK>(p, s, b, h, n, c);
}

}  // namespace bob
