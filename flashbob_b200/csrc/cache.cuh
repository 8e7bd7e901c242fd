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
#pragma once

#include "rotary.cuh"
#include "sequence.cuh"

namespace bob {

struct CacheTensor {
    uint8_t* data; long long sp, sh, sr;                         // byte strides: page, head, row
    float* scales; long long ssp, ssh, ssr;                      // 4 bits: (scale, zero) of a row; strides in floats
};

struct AppendParams {
    bob_sm100_rotary rotary;
    SequenceParams seq;
    CacheTensor cache[2];                                        // keys, values
    const uint16_t* in[2]; long long in_sb[2], in_sh[2], in_sn[2];
    int H, N, D;
};

struct ReadParams {
    SequenceParams seq;
    CacheTensor cache[2];
    uint16_t* out[2];                                            // contiguous [B, H, N, D]
    int H, N, D;
};

__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// Quantises a row of D = 16 * per_row elements, 16 of them in each of per_row neighbouring lanes (all lanes of the warp
// call this).  Every operation is rounded to nearest in fp32, so the codes are those of the formula in plain arithmetic: the
// product with the reciprocal stands for the quotient only where both round to the same code for certain.
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
    uint32_t code[2] = {0, 0};
    #pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float d = __fsub_rn(v[i], lo), q = d * inv;        // off by 3 * 2^-24 of at most 15
        float r = rintf(q);
        if (!(fabsf(fabsf(q - r) - 0.5f) > 1e-5f)) r = rintf(__fdiv_rn(d, scale));     // near a border, or no number
        code[i >> 3] |= static_cast<uint32_t>(min(max(__float2int_rn(r), 0), 15)) << (4 * (i & 7));
    }
    return make_uint2(code[0], code[1]);
}

constexpr int kCacheThreads = 256;

// One thread: 16 elements of a new row, of HPT heads (blockIdx.y), of keys and values.  BITS 4 turns the keys in 64 bits: a
// rounding that falls the other way can move an element by a whole step of the 4-bit row, 1/15 of its range.
template <int FORM, bool BF16, int BITS, int HPT>
__global__ void __launch_bounds__(kCacheThreads) append_kernel(const __grid_constant__ AppendParams p) {
    const int per_row = p.D / 16;
    const long long id = (long long)blockIdx.x * kCacheThreads + threadIdx.x, token = id / per_row;
    const int c = static_cast<int>(id % per_row);
    const int b = token < (long long)p.seq.B * p.N ? static_cast<int>(token / p.N) : -1, n = static_cast<int>(token % p.N);
    // the lanes of a row agree on everything here; those without a row stay for the shuffles
    bool there = b >= 0;
    int page = 0, position = 0;
    if (there) {
        const Sequence s = sequence_of(p.seq, b, p.N);
        if (n == 0 && c == 0 && blockIdx.y == 0 && !s.ok) report(p.seq.sticky, kStatusBadLength);
        position = s.start + n;
        there = n < s.count && position >= 0;
        if (there) {
            page = page_of(p.seq, b, position);
            if (page < 0) { report(p.seq.sticky, kStatusBadPage); there = false; }
        }
    }
    if (__ballot_sync(0xffffffffu, there) == 0) return;
    const int row = position & ((1 << p.seq.page_shift) - 1), h0 = blockIdx.y * HPT;
    const RowPlace<FORM> place(c, p.rotary.pairs);
    const RowPlace<kInterleaved> plain(c, 0);                    // 16 elements in a row
    Chunks k[HPT], v[HPT];
    #pragma unroll
    for (int i = 0; i < HPT; ++i) {
        k[i] = v[i] = Chunks{};
        if (there && h0 + i < p.H) {
            k[i] = place.load(p.in[0] + b * p.in_sb[0] + (h0 + i) * p.in_sh[0] + n * p.in_sn[0]);
            v[i] = plain.load(p.in[1] + b * p.in_sb[1] + (h0 + i) * p.in_sh[1] + n * p.in_sn[1]);
        }
    }
    using T = std::conditional_t<BITS == 4, double, float>;
    Turner<FORM, BF16, T> turn;
    turn.set(p.rotary, c, position);
    if constexpr (BITS == 16) {
        #pragma unroll
        for (int i = 0; i < HPT; ++i) {
            if (!there || h0 + i >= p.H) continue;
            auto at = [&](const CacheTensor& t) { return reinterpret_cast<uint16_t*>(t.data + page * t.sp + (h0 + i) * t.sh + row * t.sr); };
            place.store(at(p.cache[0]), turn(k[i]));
            plain.store(at(p.cache[1]), v[i]);
        }
    } else {
        __shared__ __align__(16) uint16_t stage[FORM == kScattered ? kCacheThreads * 16 : 8];
        #pragma unroll 1
        for (int i = 0; i < HPT; ++i) {
            Chunks x = turn(k[i]);
            int first = place.first, second = place.second;
            if constexpr (FORM == kScattered) {                  // the row's lanes bring its elements in order
                uint16_t* mine = stage + (threadIdx.x / per_row) * p.D;
                place.store(mine, x);
                __syncwarp();
                x.a = *reinterpret_cast<const uint4*>(mine + plain.first);
                x.b = *reinterpret_cast<const uint4*>(mine + plain.second);
                __syncwarp();
                first = plain.first;
                second = plain.second;
            }
            #pragma unroll
            for (int w = 0; w < 2; ++w) {
                float scale, zero;
                const uint2 code = quantise16<BF16>(w ? v[i] : x, per_row, scale, zero);
                if (!there || h0 + i >= p.H) continue;
                const CacheTensor& t = p.cache[w];
                uint8_t* dst = t.data + page * t.sp + (h0 + i) * t.sh + row * t.sr;
                *reinterpret_cast<uint32_t*>(dst + (w ? plain.first : first) / 2) = code.x;
                *reinterpret_cast<uint32_t*>(dst + (w ? plain.second : second) / 2) = code.y;
                if (c == 0) *reinterpret_cast<float2*>(t.scales + page * t.ssp + (h0 + i) * t.ssh + row * t.ssr) = make_float2(scale, zero);
            }
        }
    }
}

// One thread: 16 elements of a cached row, of HPT heads, of keys and values.  Rows behind a sequence become zero.
template <bool BF16, int BITS, int HPT>
__global__ void __launch_bounds__(kCacheThreads) read_kernel(const __grid_constant__ ReadParams p) {
    const int per_row = p.D / 16;
    const long long id = (long long)blockIdx.x * kCacheThreads + threadIdx.x, token = id / per_row;
    if (token >= (long long)p.seq.B * p.N) return;
    const int c = static_cast<int>(id % per_row), b = static_cast<int>(token / p.N), n = static_cast<int>(token % p.N);
    const Sequence s = sequence_of(p.seq, b, 0);
    if (n == 0 && c == 0 && blockIdx.y == 0 && __ldg(p.seq.lengths + b) != s.length) report(p.seq.sticky, kStatusBadLength);
    int page = -1;
    if (n < s.length) {
        page = page_of(p.seq, b, n);
        if (page < 0) report(p.seq.sticky, kStatusBadPage);
    }
    const int row = n & ((1 << p.seq.page_shift) - 1), h0 = blockIdx.y * HPT;
    Chunks x[HPT][2];
    #pragma unroll
    for (int i = 0; i < HPT; ++i) {
        #pragma unroll
        for (int w = 0; w < 2; ++w) {
            x[i][w] = Chunks{};
            if (page < 0 || h0 + i >= p.H) continue;
            const CacheTensor& t = p.cache[w];
            const uint8_t* src = t.data + page * t.sp + (h0 + i) * t.sh + row * t.sr;
            if constexpr (BITS == 16) {
                x[i][w].a = __ldg(reinterpret_cast<const uint4*>(src) + 2 * c);
                x[i][w].b = __ldg(reinterpret_cast<const uint4*>(src) + 2 * c + 1);
            } else {
                const uint2 code = __ldg(reinterpret_cast<const uint2*>(src) + c);
                const float2 sc = __ldg(reinterpret_cast<const float2*>(t.scales + page * t.ssp + (h0 + i) * t.ssh + row * t.ssr));
                x[i][w].a = make_uint4(code.x, code.y, __float_as_uint(sc.x), __float_as_uint(sc.y));
            }
        }
    }
    #pragma unroll
    for (int i = 0; i < HPT; ++i) {
        if (h0 + i >= p.H) continue;
        #pragma unroll
        for (int w = 0; w < 2; ++w) {
            Chunks y = x[i][w];
            if constexpr (BITS == 4) {
                const uint32_t code[2] = {y.a.x, y.a.y};
                const float scale = __uint_as_float(y.a.z), zero = __uint_as_float(y.a.w);
                float v[16];
                #pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = fmaf(static_cast<float>((code[j >> 3] >> (4 * (j & 7))) & 15u), scale, zero);
                y.a = narrow8<BF16>(v);
                y.b = narrow8<BF16>(v + 8);
            }
            uint4* dst = reinterpret_cast<uint4*>(p.out[w] + (((long long)b * p.H + h0 + i) * p.N + n) * p.D) + 2 * c;
            dst[0] = y.a;
            dst[1] = y.b;
        }
    }
}

}  // namespace bob
