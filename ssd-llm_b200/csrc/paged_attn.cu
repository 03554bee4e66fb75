// paged_attn.cu — attention of new tokens over the paged KV cache.
//
//   out[r][h] = sum_p w_p V[p][h / g],  w = softmax over p of scale * q[r][h] . K[p][h / g],
//   p in [max(0, len[r] - window), len[r]), g = n_head / n_head_kv
//
// One pass with a running maximum m and sum l (src/inference/flash_attention.rs:68-135), in base
// two: position p adds 2^(x_p - m) to l and 2^(x_p - m) V_p to the accumulator, x = score log2 e.
//
// What bounds it: a cached byte is read once (HBM) and meets g <= 8 queries, twice (K, V). At one
// byte an element and g = 8 an SM's share of HBM (23 B per cycle) needs 370 multiply-adds a cycle:
// three times what the FMA pipes give, a third of what m16n8k16 gives, so the products run on the
// tensor cores. tcgen05 would have 128 rows for 8 queries, and its accumulators would have to come
// back from TMEM for the softmax of every few positions; register accumulators fit this shape.
//
// Shape of the work: a tile is 32 positions (two of the cache's groups; one where that would leave
// too few warps: 16-bit caches at heads of 128, all at wider ones) for one unit = (row, 8 query heads
// of one KV head). Each warp streams its tiles through a ring of its own in shared memory, one bulk
// copy a tile (two for pages of 16 positions), into slots that the warp itself frees: there is no
// barrier between warps and the copies run ahead across units. (Loading fragments straight into
// registers, a tile ahead, kept too few bytes in flight; one more warp that asks for everybody's
// copies could not keep up.)
//   S^T = K Q^T : A = K (16 positions x 16 dims), B = q (8 heads)
//   O^T = V^T P^T : A = V^T (16 dims x 16 positions), B = P (8 heads), S^T transposed in between
//   by 8x8 matrix moves.
// Up to 4 query heads to a KV head (PACK): the 8 columns take two parts of each split operand, head
// h's first in column h, its second in column h + 4, added up after the product: half the matrix
// instructions (two thirds beside a bf16 cache) and half of q's registers (1 row over 131072
// positions, 32 / 8 heads, Q8_0: 80 -> 76 us; 32 rows over 4096, Q4_0: 67.6 -> 63.5; 16 rows, F16:
// 67 -> 65.5).
// All tiles of the call, rows in order, are dealt evenly to the CTAs and their warps, whatever the
// lengths, beginning a unit counting for two tiles; a unit that falls to several warps is joined in
// shared memory, one that falls to several CTAs through the workspace by the CTA that finishes last
// (partials in CTA order: the same bits every time).
//
// Measured (one B200, one layer, us a call, share of the measured HBM rate): 1 row over 131072
// positions, 64 / 8 heads of 128, Q8_0: 66 (66 %); 64 rows over 512 to 16384 positions: 148 - 161
// (73 - 79 %); 16 rows over 4096, BF16: 50 (83 %); 9 rows over 2048, 32 / 32 heads, Q4_0: 38 - 39
// (30 %: two columns of eight have work, and 8 warps an SM, each with one chain of scores, maximum,
// weights and products a tile, issue in 38 % of the cycles). Rows of one sequence do not share its
// cache: 128 rows of a prompt that end at position 4096, 64 / 8 heads: 201 (Q8_0), 266 (BF16), where
// the bytes, read once, and the products are worth some 10. In cycles, the first: 2500 until every
// warp has its share, 6500 until it has asked for its first four tiles, 15000 until the first product
// (queries and tiles arrive behind those of 148 SMs), some 85000 of tiles, 8000 after the last (12
// warps, then 18 CTAs are joined). 8-bit codes as offset bytes took 70 more instructions a group for
// their conversion; 16 positions a tile 78 us; queries held in registers before the first tile was
// asked for spilled. At heads of 128 and 8 queries, Q8_0, 12 warps leave 168 registers a thread, and
// 84 bytes of them are spilled.
//
// Precision: results are f32. Cached values are exact in the fragments' type (codes of the 8- and
// 4-bit types are small integers in f16, their scales are applied to scores and weights). The f32
// operands are split: q (scaled per head by a power of two) and the weights (relative to the
// tile's largest) into f16 hi + lo, 22 bits, or three bf16 parts, 24 bits, beside a bf16 cache. The
// f16 parts of a query end 2^-38 below the largest of its head, those of a weight 2^-38 below the
// tile's largest; weights of fewer than 13 bits, which count where a strong position's values are
// zero, and 8- and 4-bit caches' products of weights and V scales of fewer than 13 bits go through
// the tensor cores in passes of their own (kSmall and kProd below). The tensor cores truncate when
// they add, so products accumulate over at most 32 dims or 32 positions there and are added up in
// f32 registers. Scores are f32 numbers; a key that is not finite gives NaN.
#include <float.h>
#include <limits.h>

#include "paged.cuh"

namespace ssd {

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kMask8 = 0x807F807Fu;  // 8-bit codes as f16: q 2^-24 (paged.cuh)
// f16 weights: relative to the tile's largest (LIFT below); those under kSmall take another pass (so
// that each pass has 24 binades, 13 of f16's mantissa bits above its smallest number at the lower end).
constexpr float kSmall = 1.0f / 2048.0f, kSmallLog = -11.0f;
// 8- and 4-bit caches: a weight meets its position's V scales as f16 numbers too, multiplied by 2^k,
// so that each is below 2. Every product of the two other than zero is kProd or more in the pass that
// takes it: of 13 bits at least, of 22 from 2^-3 on. That holds where no scale is under kScaleLow and
// no weight under kProd / kScaleLow; else (one tile in twenty of normally distributed keys) each
// weight is looked at with its own position's scales. Where one is too small (one in some hundreds),
// a pass takes as many binades of weights as the tile's smallest scale leaves, and scales under
// 2^-kBin have passes of their own.
constexpr float kProd = 1.0f / 1024.0f, kScaleLow = 1.0f / 32.0f, kWeightLog = -5.0f;
constexpr float kNormal = 1.0f / 16384.0f;  // f16's smallest number of 11 bits
constexpr int kBin = 7;
constexpr float kBinSmall = 0.125f, kBinStep = 256.0f;  // kProd 2^kBin, 2^(kBin + 1)
// Products with q become scores within the subtraction of the tile's largest score, in one rounding;
// the largest one has a rounding of its own, a sixteenth at 2^20 and without bound above. Where it is
// larger (2^20 to infinity, as bits of its magnitude), the largest product is subtracted first.
constexpr uint32_t kLargeFrom = 0x49800000u, kLargeTo = 0x7F800000u;

template <int TYPE, int HD, bool PACK>
struct PagedCfg {
    static constexpr int NB = HD / 32;                       // blocks of 32 dims
    static constexpr bool QT = paged_quantized(TYPE);
    static constexpr int NS = TYPE == SSD_TYPE_BF16 ? 3 : 2;  // parts of an f32 operand
    static constexpr int NP = PACK ? (NS + 1) / 2 : NS;      // products of a fragment with them
    static constexpr int HEADS = PACK ? 4 : 8;               // query heads of a unit
    static constexpr int KW = TYPE == SSD_TYPE_Q8_0 ? 4 : (TYPE == SSD_TYPE_Q4_0 ? 2 : 8);  // words a block
    // Queries are scaled into [2^QLIFT, 2^(QLIFT + 1)): f16 parts as high as their range allows; bf16
    // parts have f32's range and stay so low that no finite key overflows a sum of 256 products.
    static constexpr int QLIFT = NS == 3 ? -10 : 13;
    // A new maximum rescales the accumulator only when it passes the old one by 2^LAZY. bf16 weights are
    // relative to 2^UP times the maximum when it was last raised, so at most 2^-4: sums of 16 of the
    // largest values at least are f32 numbers, and weights of scores 80 below the largest still are, of
    // 12 bits.
    static constexpr float LAZY = NS == 3 ? 2.0f : 16.0f;
    static constexpr float UP = NS == 3 ? 6.0f : 0.0f;
    // f16 weights are relative to the tile's largest, which is 2^LIFT (DOWN: the inverse): times a scale
    // below 2 and 2^(1/16), what a score may be off, it has to stay an f16 number.
    static constexpr float LIFT = QT ? 14.875f : 13.0f;
    static constexpr float DOWN = QT ? 3.3279655e-5f : 1.0f / 8192.0f;
    static constexpr int PASS = (int)LIFT;  // a pass's weights begin at 2^PASS
    static constexpr float CODE = TYPE == SSD_TYPE_Q8_0 ? 16777216.0f : 1.0f;  // code / fragment
    static constexpr int HALF = paged_half_bytes(TYPE, HD);  // bytes of a group's K, or V
    static constexpr int ROW = HD + 4;                       // floats of a head in a partial
    static constexpr int PART = HEADS * (ROW + 2) * 4;       // bytes: heads, then their m, their l
    static constexpr int GROUP = 2 * HALF;                   // bytes of a group
    static constexpr int TP = HD < 128 || (HD == 128 && QT) ? 2 : 1;  // groups of a tile
    static constexpr int TILE = TP * kPagedGroup;            // positions
    // Tiles that beginning a unit (its row, page and queries, each a trip to L2) counts for when the
    // work is dealt out: 33 rows of 1 to 2999 positions took 30.4 us at 0, 28.5 at 1, 27.6 at 2 and
    // 27.4 at 4; other shapes were best at 2.
    static constexpr int X = 2;
    // q fragments live in shared memory where that leaves registers for more warps.
    static constexpr bool QSM = QT && HD == 256;
    static constexpr int QB = QSM ? NB * NP * 512 : 0;
    // Warps (one CTA per SM): as many as registers allow (acc, and q where it is in registers, take
    // HD / 4 to HD / 2 each) while rings hold two tiles; then slots of a ring, up to 4.
    static constexpr int W = HD <= 96 ? (QT ? 12 : (HD == 64 ? 12 : 8))
                                      : (HD == 128 ? (KW == 4 ? 12 : 8) : (HD == 192 || QT ? 8 : 6));
    static constexpr int THREADS = W * 32;
    static constexpr int FIT = (216 * 1024 / W - QB) / (TP * GROUP);
    static constexpr int S = FIT < 4 ? FIT : 4;
    static_assert(S >= 2 && S * TP * GROUP >= PART && W <= 16, "ring");
    static constexpr int RING = S * TP * GROUP;  // at the end the warp's last partial
    static constexpr int SMEM = W * (QB + RING);
};

// The workspace: counters, two partials per CTA, one per warp.
constexpr int kPagedMaxWarps = 16;
__host__ __device__ constexpr size_t paged_counter_bytes(int ctas) {
    return ((size_t)ctas * 4 + 255) & ~(size_t)255;
}

__device__ __forceinline__ void ring_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
}
// Bulk copy of `bytes` (a multiple of 16, both ends 16-byte aligned) completing on bar.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
        "l"(src), "r"(bytes), "r"(bar)
        : "memory");
}
__device__ __forceinline__ bool ring_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// Waits for phase `parity` of the barrier, `tries` polls of about a microsecond at most. When they
// run out, SSD_ERR_TIMEOUT is recorded and tries becomes 1: the lane goes on (its results are
// worthless) and ends soon.
__device__ __forceinline__ void ring_wait(uint32_t bar, uint32_t parity, uint32_t& tries, int* status) {
    if (ring_try(bar, parity)) return;
    for (uint32_t it = 1; it < tries; it++)
        if (ring_try(bar, parity)) return;
    tries = 1;
    atomicExch(status, SSD_ERR_TIMEOUT);
}
__device__ __forceinline__ void ring_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t movm(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// c = a b (FIRST), or c += a b.
template <bool BF, bool FIRST>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    const float z0 = FIRST ? 0.0f : c[0], z1 = FIRST ? 0.0f : c[1];
    const float z2 = FIRST ? 0.0f : c[2], z3 = FIRST ? 0.0f : c[3];
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%10,%11,%12,%13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z0), "f"(z1),
              "f"(z2), "f"(z3));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%10,%11,%12,%13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z0), "f"(z1),
              "f"(z2), "f"(z3));
}
__device__ __forceinline__ uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
// Bits 0-3 (4-7) of both halves as the f16 numbers nibble - 8: under the exponent of 1024 the bits
// are 1024 + n (1024 + 16 n), and one packed instruction takes that back. (The masking is one
// instruction only if it is asked for as one: two constants do not fit the instruction as such.)
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t e) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(mask), "r"(e));
    return d;
}
__device__ __forceinline__ uint32_t nibble_lo(uint32_t w) {
    return h2bits(__hsub2(bits_h2(and_or(w, 0x000F000Fu, 0x64006400u)), bits_h2(0x64086408u)));
}
__device__ __forceinline__ uint32_t nibble_hi(uint32_t w) {
    return h2bits(__hfma2(bits_h2(and_or(w, 0x00F000F0u, 0x64006400u)), bits_h2(0x2C002C00u),  // 1/16
                          bits_h2(0xD480D480u)));                                             // -72
}
// (x, y) as NS parts: each the rounding of what the parts before it left.
template <int NS>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&p)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; i++) {
        if constexpr (NS == 2) {
            const __half2 h = __floats2half2_rn(x, y);
            p[i] = h2bits(h);
            x -= __low2float(h);
            y -= __high2float(h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
            p[i] = *reinterpret_cast<const uint32_t*>(&h);
            x -= __uint_as_float(p[i] << 16);
            y -= __uint_as_float(p[i] & 0xFFFF0000u);
        }
    }
}

// A lane's view of a group in a ring slot: the words of its fragments, read as they are needed.
template <int TYPE, int HD, bool PACK>
struct PagedGroup {
    using C = PagedCfg<TYPE, HD, PACK>;
    uint8_t* slot;
    int lane;
    uint32_t vs[C::QT ? 2 * C::NB : 1];  // V scales of (2t, 2t+1) for each block, then (2t+8, 2t+9)

    __device__ __forceinline__ static void words(const uint8_t* part, int b, int lane,
                                                 uint32_t (&w)[C::KW]) {
        if constexpr (C::KW == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(part + b * 256 + lane * 8);
            w[0] = x.x, w[1] = x.y;
        } else {
#pragma unroll
            for (int i = 0; i < C::KW / 4; i++) {
                const uint4 x =
                    *reinterpret_cast<const uint4*>(part + (b * (C::KW / 4) + i) * 512 + lane * 16);
                w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
            }
        }
    }
    // Fragments of K's block b: [step][register]; rows = positions g, g + 8, columns = 16 dims.
    __device__ __forceinline__ void k_frag(int b, uint32_t (&a)[2][4]) const {
        uint32_t k[C::KW];
        words(slot, b, lane, k);
#pragma unroll
        for (int s = 0; s < 2; s++) {
            if constexpr (C::KW == 8) {
                a[s][0] = k[2 * s], a[s][1] = k[4 + 2 * s];
                a[s][2] = k[2 * s + 1], a[s][3] = k[4 + 2 * s + 1];
            } else if constexpr (C::KW == 4) {
                a[s][0] = k[s] & kMask8, a[s][1] = k[2 + s] & kMask8;
                a[s][2] = __byte_perm(k[s], 0, 0x2301) & kMask8;
                a[s][3] = __byte_perm(k[2 + s], 0, 0x2301) & kMask8;
            } else {
                a[s][0] = nibble_lo(k[0] >> (8 * s)), a[s][1] = nibble_lo(k[1] >> (8 * s));
                a[s][2] = nibble_hi(k[0] >> (8 * s)), a[s][3] = nibble_hi(k[1] >> (8 * s));
            }
        }
    }
    // Scales of K's block b at positions g, g + 8.
    __device__ __forceinline__ void k_scales(float (&d)[2][C::NB]) const {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint8_t* r = slot + paged_elem_bytes(TYPE, HD) + ((lane >> 2) + 8 * i) * C::NB * 2;
            if constexpr (C::NB % 2 == 0) {
                constexpr int n = C::NB / 2;
                uint32_t w[n];
                if constexpr (n == 4) {
                    const uint4 x = *reinterpret_cast<const uint4*>(r);
                    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
                } else if constexpr (n == 2) {
                    const uint2 x = *reinterpret_cast<const uint2*>(r);
                    w[0] = x.x, w[1] = x.y;
                } else {
#pragma unroll
                    for (int j = 0; j < n; j++) w[j] = reinterpret_cast<const uint32_t*>(r)[j];
                }
#pragma unroll
                for (int j = 0; j < n; j++) {
                    const float2 f = __half22float2(bits_h2(w[j]));
                    d[i][2 * j] = f.x;
                    d[i][2 * j + 1] = f.y;
                }
            } else {
#pragma unroll
                for (int j = 0; j < C::NB; j++)
                    d[i][j] = f16_bits_to_f32(reinterpret_cast<const uint16_t*>(r)[j]);
            }
        }
    }
    // (from: where in the slot they lie)
    __device__ __forceinline__ void read_v_scales(int from) {
        if constexpr (C::QT) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint8_t* r = slot + from + ((lane & 3) + 4 * i) * C::NB * 4;
                if constexpr (C::NB % 4 == 0) {
#pragma unroll
                    for (int j = 0; j < C::NB / 4; j++) {
                        const uint4 x = reinterpret_cast<const uint4*>(r)[j];
                        uint32_t* o = vs + i * C::NB + 4 * j;
                        o[0] = x.x, o[1] = x.y, o[2] = x.z, o[3] = x.w;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < C::NB; j++)
                        vs[i * C::NB + j] = reinterpret_cast<const uint32_t*>(r)[j];
                }
            }
        }
    }
    // Clears what positions outside the tile's range hold in V (their weights are zero, but zero
    // times an infinity or a NaN is not): ok bit j: position 2t + (j & 1) + 8 (j >> 1). Scales are
    // cleared in registers, 16-bit values in the slot, each lane its own.
    __device__ __forceinline__ void mask_v(uint32_t ok) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (ok >> j & 1) continue;
#pragma unroll
            for (int b = 0; b < C::NB; b++) {
                if constexpr (C::QT)
                    vs[(j >> 1) * C::NB + b] &= j & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                else
                    *reinterpret_cast<uint2*>(slot + C::HALF + (b * 2 + (j >> 1)) * 512 + lane * 16 +
                                              (j & 1) * 8) = make_uint2(0, 0);
            }
        }
        if constexpr (!C::QT)  // before the slot's next copy
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    // V^T fragments of block b: [half s][register]; rows = dims 4g + 2s, 4g + 2s + 1, columns = 16
    // positions.
    __device__ __forceinline__ void v_frag(int b, uint32_t (&a)[2][4]) const {
        uint32_t v[C::KW];
        words(slot + C::HALF, b, lane, v);
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int p = 0; p < 2; p++) {
                if constexpr (C::KW == 8) {
                    a[s][2 * p] = __byte_perm(v[4 * p + s], v[4 * p + 2 + s], 0x5410);
                    a[s][2 * p + 1] = __byte_perm(v[4 * p + s], v[4 * p + 2 + s], 0x7632);
                } else if constexpr (C::KW == 4) {
                    a[s][2 * p] = v[2 * p + s] & kMask8;
                    a[s][2 * p + 1] = __byte_perm(v[2 * p + s], 0, 0x2301) & kMask8;
                } else {
                    a[s][2 * p] = nibble_lo(v[p] >> (8 * s));
                    a[s][2 * p + 1] = nibble_hi(v[p] >> (8 * s));
                }
            }
        }
    }
    // Smallest magnitudes other than zero of V's scales at positions 2t and 2t + 1 (8 more: p = 1), as f16
    // bits (zero: there is none). Zero is the largest 16-bit integer when 2^15 - 1 is added.
    __device__ __forceinline__ uint32_t v_scale_min(int p) const {
        uint32_t m = 0x7FFF7FFFu;
#pragma unroll
        for (int b = 0; b < C::NB; b++) m = __vmins2(m, (vs[p * C::NB + b] & 0x7FFF7FFFu) + 0x7FFF7FFFu);
        return (((m & 0xFFFFu) - 0x7FFFu) & 0xFFFFu) | (((m >> 16) - 0x7FFFu) << 16);
    }
};

// Tiles of a row, and its range of positions.
struct PagedRow {
    int seq, start, end, tile0, tiles;
};
template <int TILE>
__device__ __forceinline__ PagedRow paged_row(const PagedAttnArgs& a, int r) {
    PagedRow w;
    w.seq = a.seq ? a.seq[r] : r;
    const int cap = a.v.pages_per_seq << a.v.page_shift;  // checked to fit on the host
    w.end = (unsigned)w.seq < (unsigned)a.v.n_seq ? min(max(a.len[r], 0), cap) : 0;
    w.start = a.window > 0 ? max(0, w.end - a.window) : 0;
    w.tile0 = w.start / TILE;
    w.tiles = w.end / TILE + (w.end % TILE != 0) - w.tile0;
    return w;
}

// Writes 4 values of query head `h` of KV head `hk` at dims d.. of the row.
__device__ __forceinline__ void paged_out(const PagedAttnArgs& a, int hd, int row, int hk, int h,
                                          int d, const float4& v) {
    if (h >= a.group) return;
    store4(a.out + (int64_t)row * a.out_stride + (int64_t)(hk * a.group + h) * hd + d, v, a.out_vec);
}

// A place in the order of all tiles: rows, in a row KV heads, in a head groups of 8 query heads.
template <int TILE, int X>
struct PagedCursor {
    int r, hk, sub, tile;  // tile: of the row
    PagedRow w;
    __device__ __forceinline__ void start(const PagedAttnArgs& a, int row, const PagedRow& of, int off) {
        r = max(row, 0);
        w = of;
        if (w.tiles == 0) w.seq = 0, w.tiles = 1;
        const int ht = off / (w.tiles + X);
        tile = off - ht * (w.tiles + X) - X;
        hk = a.subs == 1 ? ht : ht / a.subs;
        sub = ht - hk * a.subs;
    }
    __device__ __forceinline__ void next_unit(const PagedAttnArgs& a) {
        tile = 0;
        if (++sub < a.subs) return;
        sub = 0;
        if (++hk < a.v.n_head_kv) return;
        hk = 0;
        do {  // a row with tiles follows; the bound holds if lengths change under the call
            r++;
            w = paged_row<TILE>(a, min(r, a.n_rows - 1));
        } while (w.tiles == 0 && r < a.n_rows);
        r = min(r, a.n_rows - 1);
        if (w.tiles == 0) w.seq = 0, w.tiles = 1;
    }
};

// Sums of x and y over the threads before this one (exclusive) and over the block, and the
// largest x. red: 3 ints per warp.
template <int W>
__device__ __forceinline__ void block_scan(int x, int y, int* red, int& px, int& py, int& sx, int& sy,
                                           int& mx) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int ix = x, iy = y, m = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, ix, o), b = __shfl_up_sync(0xffffffffu, iy, o);
        if (lane >= o) ix += a, iy += b;
        m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    __syncthreads();
    if (lane == 31) red[warp * 3] = ix, red[warp * 3 + 1] = iy, red[warp * 3 + 2] = m;
    __syncthreads();
    px = ix - x, py = iy - y, sx = 0, sy = 0, mx = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        if (w == warp) px += sx, py += sy;
        sx += red[w * 3];
        sy += red[w * 3 + 1];
        mx = max(mx, red[w * 3 + 2]);
    }
}

template <int TYPE, int HD, bool PACK>
__global__ void __launch_bounds__(PagedCfg<TYPE, HD, PACK>::THREADS, 1)
    k_paged_attn(const PagedAttnArgs a) {
    using C = PagedCfg<TYPE, HD, PACK>;
    constexpr int X = C::X, W = C::W, NB = C::NB, NS = C::NS, NP = C::NP, HEADS = C::HEADS, S = C::S;
    constexpr int NT = C::THREADS, TP = C::TP, TILE = C::TILE;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[W][S];
    __shared__ int s_red[3 * W];
    __shared__ int s_row[W], s_off[W], s_lohi[2];
    // partials of the CTA's warps, slots 2 w and 2 w + 1: where, the unit and its tiles
    __shared__ const float* e_ptr[2 * W];
    __shared__ int e_row[2 * W], e_ht[2 * W], e_us[2 * W], e_ue[2 * W];
    __shared__ int s_last[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int HT = a.v.n_head_kv * a.subs;
    if (lane < S) mbar_init(&full[warp][lane], 1);  // a warp's barriers are its own
    if (lane < 2) e_row[2 * warp + lane] = e_us[2 * warp + lane] = -1;
    fence_mbar_init();
    __syncwarp();
    pdl_wait();
    // ---- this CTA's tiles [lo, hi): equal shares, but whole units where that costs little. A unit
    // in two CTAs is joined through the workspace, about 3 us at the end of the call.
    int lo, hi, total, n_cta, quota, rest, row0, off0, s, e;
    PagedRow w0;  // the row of this warp's first tile, off0 tiles into it
    bool empty = true;     // there may be rows without tiles
    auto zeros = [&]() {  // their outputs, a share of them by each CTA
        for (int r = blockIdx.x; empty && r < a.n_rows; r += gridDim.x)
            if (paged_row<TILE>(a, r).tiles == 0)
                for (int i = tid; i < a.n_head * (HD / 4); i += NT)
                    store4(a.out + (int64_t)r * a.out_stride + 4 * i,
                           make_float4(0.0f, 0.0f, 0.0f, 0.0f), a.out_vec);
    };
    auto share = [&](int c) { return quota * c + min(c, rest); };
    auto divide = [&](int tiles, int units, int longest, bool& one_each) {  // whether whole units
        total = tiles;
        n_cta = max(1, min((int)gridDim.x, (total + W - 1) / W));  // a tile for every warp
        quota = total / n_cta;
        rest = total - quota * n_cta;
        lo = share(blockIdx.x);
        hi = share(blockIdx.x + 1);
        one_each = units <= n_cta && longest <= quota + quota / 4;  // unit number blockIdx.x
        return one_each || longest <= max(quota / 4, (TP == 1 ? 4 : 2) * W);
    };
    auto warps = [&]() {
        const int q = (hi - lo) / W, r = (hi - lo) - q * W;
        s = lo + q * warp + min(warp, r);
        e = s + q + (warp < r);
    };
    if (a.n_rows <= 32) {  // every warp finds its own, a row in each lane
        PagedRow w = {0, 0, 0, 0, 0};
        if (lane < a.n_rows) w = paged_row<TILE>(a, lane);
        const int size = w.tiles > 0 ? w.tiles + X : 0;  // of a unit
        int p = size, i = w.tiles > 0, longest = size;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, p, o), y = __shfl_up_sync(0xffffffffu, i, o);
            if (lane >= o) p += x, i += y;
            longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
        }
        const int tiles = __shfl_sync(0xffffffffu, p, 31) * HT, units = __shfl_sync(0xffffffffu, i, 31) * HT;
        const int first = (p - size) * HT, n = size * HT, unit0 = (i - (w.tiles > 0)) * HT;
        bool one_each;
        const bool whole = divide(tiles, units, longest, one_each);
        empty = units < a.n_rows * HT;
        if ((int)blockIdx.x >= n_cta) return zeros();
        if (whole) {
            auto from_unit = [&](int at) {  // the first unit that begins at tile `at` or after it
                const uint32_t has = __ballot_sync(0xffffffffu, at >= first && at < first + n);
                const int x = first + (n > 0 ? (at - first + size - 1) / size * size : 0);
                const int v = __shfl_sync(0xffffffffu, x, has ? __ffs((int)has) - 1 : 0);
                return has ? v : total;
            };
            if (one_each) {
                const int u = (int)blockIdx.x - unit0;
                const uint32_t has = __ballot_sync(0xffffffffu, w.tiles > 0 && u >= 0 && u < HT);
                const int from = has ? __ffs((int)has) - 1 : 0;
                lo = has ? __shfl_sync(0xffffffffu, first + u * size, from) : total;
                hi = has ? lo + __shfl_sync(0xffffffffu, size, from) : total;
            } else {
                lo = from_unit(lo);
                hi = from_unit(hi);
            }
            lo += X;
        }
        if (lo >= hi) return zeros();
        warps();
        const uint32_t has = __ballot_sync(0xffffffffu, s >= first && s < first + n);
        row0 = has ? __ffs((int)has) - 1 : 0;
        off0 = s - __shfl_sync(0xffffffffu, first, row0);
        w0.seq = __shfl_sync(0xffffffffu, w.seq, row0);
        w0.start = __shfl_sync(0xffffffffu, w.start, row0);
        w0.end = __shfl_sync(0xffffffffu, w.end, row0);
        w0.tile0 = __shfl_sync(0xffffffffu, w.tile0, row0);
        w0.tiles = __shfl_sync(0xffffffffu, w.tiles, row0);
    } else {  // every thread has a row; more rows are gone through again for each question
        const bool single = a.n_rows <= NT;
        int tl = 0, before, index, row_tiles, used, longest;  // a unit's; of the rows before; rows with tiles
        auto size_of = [&](int r) {  // of a unit of the row
            const int n = paged_row<TILE>(a, r).tiles;
            return n > 0 ? n + X : 0;
        };
        if (tid < a.n_rows) tl = size_of(tid);
        int n = tl, m = tl;
        for (int r = tid + NT; r < a.n_rows; r += NT) {
            const int x = size_of(r);
            n += x;
            m = max(m, x);
        }
        block_scan<W>(n, tl > 0, s_red, before, index, row_tiles, used, longest);
        if (!single) {
            int z0, z1, z2, z3;
            block_scan<W>(m, 0, s_red, z0, z1, z2, z3, longest);
            used = 0x7fffffff / HT;  // not counted
        }
        auto each_row = [&](auto f) {  // f(row, a unit's, before it, rows with tiles before it)
            if (single) {
                if (tl > 0) f(tid, tl, before, index);
                return;
            }
            int p0 = 0, i0 = 0;
            for (int r0 = 0; r0 < a.n_rows; r0 += NT) {
                const int x = r0 + tid < a.n_rows ? size_of(r0 + tid) : 0;
                int p, i, sp, si, z;
                block_scan<W>(x, x > 0, s_red, p, i, sp, si, z);
                if (x > 0) f(r0 + tid, x, p0 + p, i0 + i);
                p0 += sp;
                i0 += si;
            }
        };
        bool one_each;
        const bool whole = divide(row_tiles * HT, used * HT, longest, one_each);
        empty = !single || used < a.n_rows;
        if ((int)blockIdx.x >= n_cta) return zeros();
        if (whole) {
            if (tid < 2) s_lohi[tid] = total;
            __syncthreads();
            each_row([&](int, int x, int p, int i) {
                const int first = p * HT;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    if (one_each) {
                        const int u = (int)blockIdx.x - i * HT;
                        if (u >= 0 && u < HT) s_lohi[k] = first + (u + k) * x;
                    } else {  // from the first unit that begins at the share's start or after it
                        const int at = (k ? hi : lo) - first;
                        if (at >= 0 && at < x * HT) s_lohi[k] = first + (at + x - 1) / x * x;
                    }
                }
            });
            __syncthreads();
            lo = s_lohi[0] + X;
            hi = s_lohi[1];
        }
        if (lo >= hi) return zeros();
        warps();
        if (lane == 0) s_row[warp] = 0;
        __syncthreads();
        each_row([&](int r, int x, int p, int) {  // the row of each warp's first tile
            const int first = p * HT, q = (hi - lo) / W, left = (hi - lo) - q * W;
            if (first >= hi || first + x * HT <= lo) return;
            for (int w = 0; w < W; w++) {
                const int at = lo + q * w + min(w, left) - first;
                if (at >= 0 && at < x * HT) {
                    s_row[w] = r;
                    s_off[w] = at;
                }
            }
        });
        __syncthreads();
        row0 = s_row[warp];
        off0 = s_off[warp];
        w0 = paged_row<TILE>(a, row0);
    }

    // partials: a CTA's two (units that other CTAs hold too), a warp's first; its last is in its ring
    // part k of a split operand for this lane's column: where parts are packed, head g % 4's part
    // 2 k + g / 4
    auto part_of = [&](const uint32_t(&p)[NS], int k) -> uint32_t {
        if constexpr (!PACK) return p[k];
        if (2 * k + 1 < NS) return g < 4 ? p[2 * k] : p[min(2 * k + 1, NS - 1)];
        return g < 4 ? p[2 * k] : 0u;
    };
    uint32_t* counters = reinterpret_cast<uint32_t*>(a.work);
    const size_t part_f = C::PART / 4;
    float* parts = reinterpret_cast<float*>(a.work + paged_counter_bytes(gridDim.x));
    auto warp_part = [&](int w) {
        return parts + (2 * (size_t)gridDim.x + (size_t)blockIdx.x * W + w) * part_f;
    };
    if (s < e) {
        uint8_t* qsm = smem + warp * (C::QB + C::RING);  // q fragments
        uint8_t* ring = qsm + C::QB;                     // its slots; then its last partial
        const uint32_t full0 = smem_u32(&full[warp][0]), ring0 = smem_u32(ring);
        PagedCursor<TILE, C::X> cur;
        cur.start(a, row0, w0, off0);
        if (cur.tile < 0) s -= cur.tile, cur.tile = 0;
        // ---- the copies: `ahead` is the next tile to ask for, src0 and src1 where its groups lie
        // (null: no page)
        constexpr int G = C::GROUP;
        const bool paired = TP == 1 || a.v.page_shift > 4;  // a page holds whole tiles
        const int page_tiles = paired ? a.v.page_shift - 3 - TP : 0, page_mask = (1 << page_tiles) - 1;
        PagedCursor<TILE, C::X> ahead = cur;
        int left = e - s;         // tiles not asked for yet, and beginnings of units
        uint32_t missing = 0;     // bits 2 i, 2 i + 1: the groups of slot i that have no page
        const uint8_t *src0, *src1;
        int ids = -1, ids0 = INT_MIN / 2;  // lane i: the sequence's page ids0 + i
        auto page = [&](int i) -> const uint8_t* {  // i-th page of the row's sequence
            if ((unsigned)(i - ids0) >= 32u) {
                ids0 = i;
                ids = i + lane < a.v.pages_per_seq
                          ? a.v.table[(size_t)ahead.w.seq * a.v.pages_per_seq + i + lane]
                          : -1;
            }
            const int id = __shfl_sync(0xffffffffu, ids, i - ids0);
            return (unsigned)id < (unsigned)a.v.n_pages
                       ? a.v.pool + (uint64_t)id * a.v.page_bytes + (size_t)ahead.hk * a.v.head_bytes
                       : nullptr;
        };
        auto enter = [&](int i) {  // tile i of the sequence, in another page than the one before
            if (paired) {
                src0 = page(i >> page_tiles);
                if (src0) src0 += (size_t)(i & page_mask) * (TP * G);
                src1 = src0 ? src0 + G : nullptr;
            } else {
                src0 = page(2 * i);
                src1 = page(2 * i + 1);
            }
        };
        // The unit's queries into L2 before its tiles are asked for: loads of them from HBM would
        // queue behind those of every SM.
        auto want_q = [&]() {
            const int h = ahead.sub * HEADS + g % HEADS;
            if (h >= a.group) return;
            const float* q = a.q + (int64_t)ahead.r * a.q_stride + (int64_t)(ahead.hk * a.group + h) * HD;
            for (int i = t; i < NB; i += 4) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + 32 * i));
        };
        auto ask = [&](int slot) {
            if (left <= 0) return;
            missing = (missing & ~(3u << 2 * slot)) | ((src0 ? 0u : 1u) | (src1 ? 0u : 2u)) << 2 * slot;
            if (lane == 0) {
                const uint32_t bar = full0 + slot * 8, dst = ring0 + slot * TP * G;
                const uint32_t n = (src0 ? G : 0) + (TP == 2 && src1 ? G : 0);
                if (n)
                    ring_expect(bar, n);
                else
                    ring_arrive(bar);
                if (paired) {
                    if (src0) bulk_load(dst, src0, TP * G, bar);
                } else {
                    if (src0) bulk_load(dst, src0, G, bar);
                    if (src1) bulk_load(dst + G, src1, G, bar);
                }
            }
            if (--left <= 0) return;
            if (++ahead.tile == ahead.w.tiles) {
                if ((left -= X) <= 0) return;
                const int seq = ahead.w.seq;
                ahead.next_unit(a);
                if (ahead.w.seq != seq) ids0 = INT_MIN / 2;
                want_q();
                enter(ahead.w.tile0);
                return;
            }
            const int i = ahead.w.tile0 + ahead.tile;
            if ((i & page_mask) == 0)
                enter(i);
            else if (src0)
                src0 += TP * G, src1 += TP * G;
        };
        if (left > 0) {
            want_q();
            enter(ahead.w.tile0 + ahead.tile);
        }
#pragma unroll 1
        for (int i = 0; i < S; i++) ask(i);
        int slot = 0;
        uint32_t phase = 0;
        bool first_piece = true;
        uint32_t tries = 1u << 20;
        while (s < e) {
            const PagedRow& rw = cur.w;
            const int tile = cur.tile, r = cur.r, hk = cur.hk, h0 = cur.sub * HEADS;
            const int n = min(rw.tiles - tile, e - s);
            // ---- q fragments of the unit's heads, head g's scaled into [2^QLIFT, 2^(QLIFT + 1))
            float c1;
            uint32_t qf[C::QSM ? 1 : NB][NP][4];  // step s, register i: 2 s + i
            uint4* qs = reinterpret_cast<uint4*>(qsm) + lane;
            {
                const int h = h0 + g % HEADS;
                const bool has = h < a.group;
                const float* q = a.q + (int64_t)r * a.q_stride +
                                 (int64_t)(hk * a.group + (has ? h : h0)) * HD + 8 * t;
                float amax = 0.0f;
                float x[NB][8];
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const float4 y = load4(q + 32 * b, a.q_vec), z = load4(q + 32 * b + 4, a.q_vec);
                    x[b][0] = y.x, x[b][1] = y.y, x[b][2] = y.z, x[b][3] = y.w;
                    x[b][4] = z.x, x[b][5] = z.y, x[b][6] = z.z, x[b][7] = z.w;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        x[b][i] = has ? x[b][i] : 0.0f;
                        amax = fmaxf(amax, fabsf(x[b][i]));
                    }
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                int ex = (int)(__float_as_uint(amax) >> 23);
                // (largest queries below 2^-113: less; beside a bf16 cache above 2^60: down by 2^70)
                ex = ex == 255 ? 127 : min(max(ex, 14), NS == 3 ? 187 : 254);
                const float up = __uint_as_float((uint32_t)(254 + C::QLIFT - ex) << 23);
                c1 = fmaxf(__uint_as_float((uint32_t)(ex - C::QLIFT) << 23) * a.scale * kLog2e * C::CODE, FLT_MIN);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint32_t(&f)[NP][4] = qf[C::QSM ? 0 : b];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int d0 = TYPE == SSD_TYPE_Q4_0 ? i : 2 * i;
                        const int d1 = TYPE == SSD_TYPE_Q4_0 ? i + 4 : 2 * i + 1;
                        uint32_t p[NS];
                        split_pair<NS>(x[b][d0] * up, x[b][d1] * up, p);
#pragma unroll
                        for (int k = 0; k < NP; k++) f[k][i] = part_of(p, k);
                    }
                    if constexpr (C::QSM) {  // read back by the lane that wrote it
#pragma unroll
                        for (int k = 0; k < NP; k++)
                            qs[(b * NP + k) * 32] = make_uint4(f[k][0], f[k][1], f[k][2], f[k][3]);
                    }
                }
            }
            // ---- the tiles
            float acc[NB][2][4];
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[b][i][j] = 0.0f;
            float m = -INFINITY, l = 0.0f;  // of head g (m with UP)
            // V's scales are multiplied by 2^k (dk: twice, as f16), the products with P by 2^-k DOWN (unlift)
            uint32_t dk = 0x78007800u, scale_low = 0x00100010u;  // k = 15; kScaleLow 2^-k
            float unlift = C::QT ? C::CODE * C::DOWN / 32768.0f : C::DOWN;
            for (int i = 0; i < n; i++) {
                ring_wait(full0 + slot * 8, phase, tries, a.status);
                PagedGroup<TYPE, HD, PACK> T[TP];
                float x[TP][4];  // products of head g at positions 2t, 2t+1, 2t+8, 2t+9; times c1: scores
#pragma unroll
                for (int j = 0; j < TP; j++) {
                    T[j].slot = ring + (slot * TP + j) * G;
                    T[j].lane = lane;
                }
                const int p0 = (rw.tile0 + tile + i) * TILE;
                const uint32_t miss = missing >> 2 * slot & 3u;
                auto inside = [&](int j) {  // of the lane's positions of group j
                    uint32_t ok = 0;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int p = p0 + 16 * j + 2 * t + (k & 1) + 8 * (k >> 1);
                        if (!(miss >> j & 1) && p >= rw.start && p < rw.end) ok |= 1u << k;
                    }
                    return ok;
                };
                const bool part = miss || p0 < rw.start || rw.end - p0 < TILE;
                // The tile's V scales as 32-bit words (two positions of a block), in the order of pairs,
                // then blocks: the lane's share of them, without those of positions outside the range.
                constexpr int WORDS = NB * 8, SHARE = (TP * WORDS + 31) / 32;
                auto word_of = [&](int i) {  // (some lanes: one twice)
                    const int at = i * 32 + lane;
                    return at < TP * WORDS ? at : lane;
                };
                auto word_at = [&](int at, int of) {  // of: C::HALF, or 0: in the place of K's scales
                    const int j = at / WORDS;
                    return reinterpret_cast<uint32_t*>(T[0].slot + j * G + of + paged_elem_bytes(TYPE, HD)) +
                           (at - j * WORDS);
                };
                auto scales = [&](int i) -> uint32_t {
                    const int at = word_of(i), j = at / WORDS, p = p0 + 16 * j + 2 * ((at - j * WORDS) / NB);
                    uint32_t d = *word_at(at, C::HALF);
                    if (part && ((miss >> j & 1) || p < rw.start || p >= rw.end)) d &= 0xFFFF0000u;
                    if (part && ((miss >> j & 1) || p + 1 < rw.start || p + 1 >= rw.end)) d &= 0x0000FFFFu;
                    return d;
                };
                bool odd = part;  // a scale, times 2^k, may be 2 or more or under kScaleLow
                __half2 hi, lo;
                if constexpr (C::QT) {
#pragma unroll
                    for (int i = 0; i < SHARE; i++) {
                        uint32_t d = *word_at(word_of(i), C::HALF);
                        if constexpr (TYPE == SSD_TYPE_Q4_0) d &= 0x7FFF7FFFu;
                        hi = i ? __hmax2(hi, bits_h2(d)) : bits_h2(d);
                        lo = i ? __hmin2(lo, bits_h2(d)) : bits_h2(d);
                    }
                    odd |= !__hblt2(hi, bits_h2(0x7C007C00u - dk)) || !__hbge2(lo, bits_h2(scale_low));
                }
                // Q K
                {
                    float kd[TP][2][C::QT ? NB : 1];
                    float S4[TP][4];
#pragma unroll
                    for (int j = 0; j < TP; j++) {
                        if constexpr (C::QT) T[j].k_scales(kd[j]);
#pragma unroll
                        for (int k = 0; k < 4; k++) S4[j][k] = 0.0f;
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        uint32_t q[NP][4];
#pragma unroll
                        for (int k = 0; k < NP; k++) {
                            if constexpr (C::QSM) {
                                const uint4 y = qs[(b * NP + k) * 32];
                                q[k][0] = y.x, q[k][1] = y.y, q[k][2] = y.z, q[k][3] = y.w;
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; j++) q[k][j] = qf[b][k][j];
                            }
                        }
#pragma unroll
                        for (int j = 0; j < TP; j++) {
                            float c[4];
                            uint32_t f[2][4];
                            T[j].k_frag(b, f);
                            mma16816<NS == 3, true>(c, f[0], q[0][0], q[0][1]);
                            mma16816<NS == 3, false>(c, f[1], q[0][2], q[0][3]);
#pragma unroll
                            for (int k = 1; k < NP; k++) {
                                mma16816<NS == 3, false>(c, f[0], q[k][0], q[k][1]);
                                mma16816<NS == 3, false>(c, f[1], q[k][2], q[k][3]);
                            }
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                S4[j][k] = C::QT ? fmaf(kd[j][k >> 1][C::QT ? b : 0], c[k], S4[j][k])
                                                 : S4[j][k] + c[k];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < TP; j++)
#pragma unroll
                        for (int p = 0; p < 2; p++) {
                            const uint32_t s0 = __float_as_uint(S4[j][2 * p]);
                            const uint32_t s1 = __float_as_uint(S4[j][2 * p + 1]);
                            const uint32_t l16 = movm(__byte_perm(s0, s1, 0x5410));
                            const uint32_t h16 = movm(__byte_perm(s0, s1, 0x7632));
                            x[j][2 * p] = __uint_as_float(__byte_perm(l16, h16, 0x5410));
                            x[j][2 * p + 1] = __uint_as_float(__byte_perm(l16, h16, 0x7632));
                            if constexpr (PACK) {
                                x[j][2 * p] += __shfl_xor_sync(0xffffffffu, x[j][2 * p], 16);
                                x[j][2 * p + 1] += __shfl_xor_sync(0xffffffffu, x[j][2 * p + 1], 16);
                            }
                        }
                }
#pragma unroll
                for (int j = 0; j < TP; j++) T[j].read_v_scales(C::HALF + paged_elem_bytes(TYPE, HD));
                if (part) {
#pragma unroll
                    for (int j = 0; j < TP; j++) {
                        const uint32_t ok = inside(j);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            if (!(ok >> k & 1)) x[j][k] = -INFINITY;
                        T[j].mask_v(ok);
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < TP; j++)
                    mx = fmaxf(mx, fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])));
                if constexpr (NS == 2) {  // the tile's largest score of head g
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                }
                mx *= c1;
                // weights are 2^(x c1 - base): relative to the tile's largest, or to m
                float base = NS == 3 ? (m == -INFINITY ? 0.0f : m) : (mx == -INFINITY ? 0.0f : mx - C::LIFT);
                const bool large = (__float_as_uint(mx) & 0x7FFFFFFFu) - kLargeFrom < kLargeTo - kLargeFrom;
                bool update = mx > m + (C::LAZY - C::UP) || large, again = false;
                if constexpr (NS == 2) {
                    float mn = INFINITY;
#pragma unroll
                    for (int j = 0; j < TP; j++)
                        mn = fminf(mn, fminf(fminf(x[j][0], x[j][1]), fminf(x[j][2], x[j][3])));
                    const float low = fmaf(mn, c1, -base);  // log2 of the lane's smallest weight
                    again = low < (C::QT ? kWeightLog : kSmallLog);
                }
                if (__any_sync(0xffffffffu, update || again || (C::QT && odd))) {
                    if constexpr (C::QT) {
                        if (__any_sync(0xffffffffu, odd)) {  // 2^k for this tile: its largest scale to [1, 2)
                            uint32_t top = 0;
#pragma unroll
                            for (int i = 0; i < SHARE; i++) {
                                const uint32_t d = scales(i) & 0x7FFF7FFFu;
                                top = max(top, max(d & 0xFFFFu, d >> 16));
                            }
                            const int e = max(30 - (int)(__reduce_max_sync(0xffffffffu, top) >> 10), 0);  // k + 15
                            dk = e ? (uint32_t)e * 0x04000400u : 0x02000200u;
                            const float down = __uint_as_float((uint32_t)(142 - e) << 23);  // 2^-k
                            unlift = down * (C::CODE * C::DOWN);
                            scale_low = __half_as_ushort(__float2half_rn(kScaleLow * down)) * 0x10001u;
                            again |= part || !__hbge2(lo, bits_h2(scale_low));
                        }
                    }
                    again = __any_sync(0xffffffffu, again);
                    if constexpr (NS == 3) {
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    }
                    if (__any_sync(0xffffffffu, update)) {
                        const float mn = fmaxf(m, mx + C::UP);
                        const float f = m == -INFINITY ? 0.0f : ex2(m - mn);
                        m = mn;
                        if constexpr (NS == 3) base = m == -INFINITY ? 0.0f : m;
                        l *= f;
                        const float f0 = __shfl_sync(0xffffffffu, f, 8 * t);
                        const float f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
                        for (int b = 0; b < NB; b++)
#pragma unroll
                            for (int i = 0; i < 2; i++)
#pragma unroll
                                for (int j = 0; j < 4; j++) acc[b][i][j] *= j & 1 ? f1 : f0;
                        if (__any_sync(0xffffffffu, large)) {
                            float top = -INFINITY;
#pragma unroll
                            for (int j = 0; j < TP; j++)
                                top = fmaxf(top, fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                            if (top > -INFINITY) {
                                base = NS == 3 ? m - mx : -C::LIFT;
#pragma unroll
                                for (int j = 0; j < TP; j++)
#pragma unroll
                                    for (int k = 0; k < 4; k++) x[j][k] -= top;
                            }
                            again = NS == 2;
                        }
                    }
                }
                float w[TP][4], fa = 1.0f, fb = 1.0f;  // weights; what P V of heads 2t, 2t+1 counts
#pragma unroll
                for (int j = 0; j < TP; j++)
#pragma unroll
                    for (int k = 0; k < 4; k++) w[j][k] = ex2(fmaf(x[j][k], c1, -base));
                float sum = (w[0][0] + w[0][1]) + (w[0][2] + w[0][3]);
                if constexpr (TP == 2) sum += (w[TP - 1][0] + w[TP - 1][1]) + (w[TP - 1][2] + w[TP - 1][3]);
                if constexpr (NS == 2) {
                    const float beta = m == -INFINITY ? 0.0f : ex2(mx - m);
                    l = fmaf(sum, beta * C::DOWN, l);
                    fa = __shfl_sync(0xffffffffu, beta, 8 * t) * unlift;
                    fb = __shfl_sync(0xffffffffu, beta, 8 * t + 4) * unlift;
                } else {
                    l += sum;
                }
                // P V; for f16 weights in as many passes as their range needs (one, as a rule; the others
                // in a copy of the code, which leaves the rule's without a loop)
                auto products = [&](const float (&u)[TP][4]) {
                    uint32_t pu[TP][2][NS];
#pragma unroll
                    for (int j = 0; j < TP; j++)
#pragma unroll
                        for (int p = 0; p < 2; p++)
                            split_pair<NS>(u[j][2 * p], u[j][2 * p + 1], pu[j][p]);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        uint32_t pb[TP][2][NP], f[TP][2][4];
#pragma unroll
                        for (int j = 0; j < TP; j++) {
                            T[j].v_frag(b, f[j]);
#pragma unroll
                            for (int p = 0; p < 2; p++) {
                                if constexpr (C::QT) {  // (hi + lo) d, the low part by the residual
                                    const __half2 d =
                                        __hmul2(bits_h2(T[j].vs[p * NB + b]), bits_h2(dk));
                                    const __half2 hi = bits_h2(pu[j][p][0]), h = __hmul2(hi, d);
                                    const __half2 r = __hfma2(hi, d, __hneg2(h));
                                    const uint32_t parts[2] = {
                                        h2bits(h), h2bits(__hfma2(bits_h2(pu[j][p][1]), d, r))};
#pragma unroll
                                    for (int k = 0; k < NP; k++) pb[j][p][k] = part_of(parts, k);
                                } else {
#pragma unroll
                                    for (int k = 0; k < NP; k++) pb[j][p][k] = part_of(pu[j][p], k);
                                }
                            }
                        }
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            float c[4];
                            mma16816<NS == 3, true>(c, f[0][h], pb[0][0][0], pb[0][1][0]);
#pragma unroll
                            for (int k = 1; k < NP; k++)
                                mma16816<NS == 3, false>(c, f[0][h], pb[0][0][k], pb[0][1][k]);
#pragma unroll
                            for (int k = 0; TP == 2 && k < NP; k++)
                                mma16816<NS == 3, false>(c, f[TP - 1][h], pb[TP - 1][0][k], pb[TP - 1][1][k]);
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                acc[b][h][k] = NS == 2 ? fmaf(c[k], k & 1 ? fb : fa, acc[b][h][k])
                                                       : acc[b][h][k] + c[k];
                        }
                    }
                };
                const float up = __uint_as_float(((dk >> 26) + 112) << 23);  // 2^k
                if (NS == 2 && again) {
                    again = false;
#pragma unroll
                    for (int j = 0; j < TP; j++)
#pragma unroll
                        for (int p = 0; p < 2; p++) {
                            uint32_t least = 0;
                            if constexpr (C::QT) least = T[j].v_scale_min(p);
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const float d = f16_bits_to_f32((uint16_t)(least >> 16 * k)) * up, y = w[j][2 * p + k];
                                again |= y > 0.0f && (C::QT ? d > 0.0f && (y * d < kProd || d < kNormal) : y < kSmall);
                            }
                        }
                    again = __any_sync(0xffffffffu, again);
                }
                if (NS == 3 || !again) {
                    products(w);
                } else {
                    float small = kSmall;  // a pass takes weights down to this
                    if constexpr (C::QT) {
                        uint32_t least = 0x7800u;  // f16 bits of the smallest scale other than zero, less one
#pragma unroll
                        for (int i = 0; i < SHARE; i++) {
                            const uint32_t d = scales(i) & 0x7FFF7FFFu;
                            least = min(least, min((d & 0xFFFFu) - 1u, (d >> 16) - 1u));
                        }
                        least = __reduce_min_sync(0xffffffffu, least);
                        const int e = (int)(__float_as_uint(f16_bits_to_f32((uint16_t)least) * up) >> 23);
                        small = e < 127 - kBin ? kBinSmall : kProd * __uint_as_float((uint32_t)(254 - e) << 23);
                    }
                    float by = 1.0f;  // the pass's factor on the scales
                    do {
                        float u[TP][4], next;  // fa, fb to the next pass's
                        bool rest = false;     // smaller scales have to meet the same weights
                        if constexpr (C::QT) {
                            if (small == kBinSmall) {  // this pass's scales, in the place of K's
                                constexpr float from = 1.0f / (1 << kBin);
                                const float to = by == 1.0f ? NAN : from * kBinStep;  // (the first: all above)
                                __syncwarp();
#pragma unroll
                                for (int i = 0; i < SHARE; i++) {
                                    const float2 d = __half22float2(bits_h2(scales(i)));
                                    const float y = fabsf(d.x) * (up * by), z = fabsf(d.y) * (up * by);
                                    rest |= (y > 0.0f && y < from) || (z > 0.0f && z < from);
                                    *word_at(word_of(i), 0) =
                                        h2bits(__floats2half2_rn(y < from || y >= to ? 0.0f : d.x * by,
                                                                 z < from || z >= to ? 0.0f : d.y * by));
                                }
                                rest = __any_sync(0xffffffffu, rest);
                                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // as mask_v
                                __syncwarp();
#pragma unroll
                                for (int j = 0; j < TP; j++) T[j].read_v_scales(paged_elem_bytes(TYPE, HD));
                            }
                        }
                        const float step = __uint_as_float(((uint32_t)(254 + C::PASS) << 23) - __float_as_uint(small));
                        again = false;
#pragma unroll
                        for (int j = 0; j < TP; j++)
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const bool later = w[j][k] < small;
                                again |= later && w[j][k] > 0.0f;
                                u[j][k] = later ? 0.0f : w[j][k];
                                if (!rest) w[j][k] = later ? w[j][k] * step : 0.0f;
                            }
                        again = rest || __any_sync(0xffffffffu, again);
                        next = rest ? 1.0f / kBinStep : by * (small / (1 << C::PASS));
                        by = rest ? by * kBinStep : 1.0f;
                        products(u);
                        fa *= next;
                        fb *= next;
                    } while (again);
                }
                __syncwarp();  // the slot is read
                ask(slot);
                if (++slot == S) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            // ---- this piece: the unit's output if it is the whole unit, else a partial
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if constexpr (PACK) {
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            acc[b][i][j] += __shfl_xor_sync(0xffffffffu, acc[b][i][j], 2);
            }
            if (tile == 0 && n == rw.tiles) {
                const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
                const float i0 = __shfl_sync(0xffffffffu, inv, 8 * t);
                const float i1 = __shfl_sync(0xffffffffu, inv, 8 * t + 4);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const float(&c)[2][4] = acc[b];
                    paged_out(a, HD, r, hk, h0 + 2 * t, 32 * b + 4 * g,
                              make_float4(c[0][0] * i0, c[0][2] * i0, c[1][0] * i0, c[1][2] * i0));
                    paged_out(a, HD, r, hk, h0 + 2 * t + 1, 32 * b + 4 * g,
                              make_float4(c[0][1] * i1, c[0][3] * i1, c[1][1] * i1, c[1][3] * i1));
                }
            } else {
                const int at = 2 * warp + (first_piece ? 0 : 1);
                // a warp's last piece may use its ring, which is done
                float* o = s + n == e ? reinterpret_cast<float*>(ring) : warp_part(warp);
                __syncwarp();
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const float(&c)[2][4] = acc[b];
                    if (2 * t >= HEADS) break;
                    *reinterpret_cast<float4*>(o + 2 * t * C::ROW + 32 * b + 4 * g) =
                        make_float4(c[0][0], c[0][2], c[1][0], c[1][2]);
                    *reinterpret_cast<float4*>(o + (2 * t + 1) * C::ROW + 32 * b + 4 * g) =
                        make_float4(c[0][1], c[0][3], c[1][1], c[1][3]);
                }
                if (t == 0 && g < HEADS) {
                    o[HEADS * C::ROW + g] = m;
                    o[HEADS * (C::ROW + 1) + g] = l;
                }
                if (lane == 0) {
                    e_ptr[at] = o;
                    e_row[at] = r;
                    e_ht[at] = hk * a.subs + cur.sub;
                    e_us[at] = s - tile;
                    e_ue[at] = s - tile + rw.tiles;
                }
            }
            first_piece = false;
            s += tile + n == rw.tiles ? n + X : n;
            if (s < e) cur.next_unit(a);
        }
        if (tries == 1)  // a wait gave up: let the copies that were asked for end before the CTA does
            for (int i = 0; i < S; i++) {
                mbar_wait(&full[warp][i], 0, nullptr);
                mbar_wait(&full[warp][i], 1, nullptr);
            }
    }
    zeros();
    __syncthreads();

    // ---- join partials, first the CTA's of each unit it holds (slots in order: warps in order),
    // then, of each unit of several CTAs, theirs (in order, by the last of them to come here). One
    // loop for both: most of the time here goes into fetching instructions.
    constexpr int ITEMS = HEADS * (HD / 4);  // a unit's outputs in fours
    constexpr uint32_t kSlots = 0xffffffffu >> (32 - 2 * W);
    uint32_t held = __ballot_sync(0xffffffffu, e_row[min(lane, 2 * W - 1)] >= 0) & kSlots;
    int open_c0[2] = {-1, -1}, open_c1[2] = {-1, -1}, open_row[2] = {0, 0}, open_ht[2] = {0, 0};
    int k = -1;  // of the CTA's own: -1; then which of the two open units
#pragma unroll 1
    while (true) {
        uint32_t mine = 0;  // slots
        int n, row, ht, c0 = 0, part_k = 0;
        bool whole = true;
        if (held) {
            const int x0 = __ffs((int)held) - 1, us = e_us[x0], ue = e_ue[x0];
            mine = __ballot_sync(0xffffffffu, e_us[min(lane, 2 * W - 1)] == us) & held;
            held &= ~mine;
            n = __popc(mine);
            row = e_row[x0];
            ht = e_ht[x0];
            whole = us >= lo && ue <= hi;
            if (!whole) {  // CTAs c0 .. c1 hold it
                auto cta_of = [&](int x) {
                    const int big = rest * (quota + 1);
                    return x < big ? x / (quota + 1) : rest + (x - big) / max(quota, 1);
                };
                const int first = cta_of(us), last = cta_of(ue - 1);
                part_k = us >= lo;  // it begins here, or came from the CTA before
#pragma unroll
                for (int j = 0; j < 2; j++)
                    if (j == part_k)
                        open_c0[j] = first, open_c1[j] = last, open_row[j] = row, open_ht[j] = ht;
            }
        } else {
            if (k < 0) {
                if (open_c0[0] < 0 && open_c0[1] < 0) return;
                __threadfence();
                __syncthreads();
                if (tid < 2) {
                    const int b = tid ? open_c0[1] : open_c0[0], c = tid ? open_c1[1] : open_c1[0];
                    s_last[tid] = b >= 0 && atomicAdd(&counters[b], 1u) == (uint32_t)(c - b);
                }
                __syncthreads();
                __threadfence();
            }
            if (++k == 2) return;
            if (!s_last[k]) continue;
            c0 = k ? open_c0[1] : open_c0[0];
            n = (k ? open_c1[1] : open_c1[0]) - c0 + 1;
            row = k ? open_row[1] : open_row[0];
            ht = k ? open_ht[1] : open_ht[0];
            if (tid == 0) counters[c0] = 0;
        }
        float* part = parts + ((size_t)blockIdx.x * 2 + part_k) * part_f;
#pragma unroll 1
        for (int i = tid; i < ITEMS; i += NT) {
            const int h = i / (HD / 4), d = i % (HD / 4) * 4;
            float M = -INFINITY, L = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            constexpr int AT = 6;  // partials in flight
            uint32_t slots = mine;
#pragma unroll 1
            for (int c = 0; c < n; c += AT) {
                float m[AT], l[AT];
                float4 v[AT];
                float mn = M;
#pragma unroll
                for (int j = 0; j < AT; j++) {
                    m[j] = -INFINITY, l[j] = 0.0f, v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (c + j < n) {
                        // CTA c0's is its second, the others' their first. Plain loads: the fences
                        // around the counter order them (relaxed ones took 1 to 4 % of a call).
                        const float* p = k < 0 ? e_ptr[__ffs((int)slots) - 1]
                                               : parts + ((size_t)(c0 + c + j) * 2 + (c + j == 0)) * part_f;
                        slots &= slots - 1;
                        m[j] = p[HEADS * C::ROW + h];
                        l[j] = p[HEADS * (C::ROW + 1) + h];
                        v[j] = *reinterpret_cast<const float4*>(p + h * C::ROW + d);
                    }
                }
#pragma unroll
                for (int j = 0; j < AT; j++) mn = fmaxf(mn, m[j]);
                const float base = mn == -INFINITY ? 0.0f : mn;
                const float f0 = ex2(M - base);
                M = mn;
                L *= f0;
                o = make_float4(o.x * f0, o.y * f0, o.z * f0, o.w * f0);
#pragma unroll
                for (int j = 0; j < AT; j++) {
                    const float f = ex2(m[j] - base);
                    L = fmaf(l[j], f, L);
                    o.x = fmaf(v[j].x, f, o.x);
                    o.y = fmaf(v[j].y, f, o.y);
                    o.z = fmaf(v[j].z, f, o.z);
                    o.w = fmaf(v[j].w, f, o.w);
                }
            }
            if (whole) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
                paged_out(a, HD, row, ht / a.subs, ht % a.subs * HEADS + h, d, o);
            } else {
                *reinterpret_cast<float4*>(part + h * C::ROW + d) = o;
                if (d == 0) {
                    part[HEADS * C::ROW + h] = M;
                    part[HEADS * (C::ROW + 1) + h] = L;
                }
            }
        }
    }
}

struct AttnLaunch {
    ssd_ctx* ctx;
    const PagedAttnArgs& a;
    cudaStream_t s;
    bool pdl;
    template <int TYPE, int HD>
    int run() const {
        return a.group <= 4 ? go<TYPE, HD, true>() : go<TYPE, HD, false>();
    }
    template <int TYPE, int HD, bool PACK>
    int go() const {
        using C = PagedCfg<TYPE, HD, PACK>;
        const int grid = ctx->num_sms;
        SSD_CK(launch_pdl(k_paged_attn<TYPE, HD, PACK>, dim3(grid), dim3(C::THREADS), C::SMEM, s, pdl, a));
        return SSD_OK;
    }
};

struct AttnLoad {
    template <int TYPE, int HD>
    int run() const {
        SSD_TRY((go<TYPE, HD, true>()));
        return go<TYPE, HD, false>();
    }
    template <int TYPE, int HD, bool PACK>
    static int go() {
        cudaFuncAttributes at;
        SSD_CK(cudaFuncGetAttributes(&at, k_paged_attn<TYPE, HD, PACK>));
        SSD_CK(cudaFuncSetAttribute(k_paged_attn<TYPE, HD, PACK>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    PagedCfg<TYPE, HD, PACK>::SMEM));
        return SSD_OK;
    }
};
int load_paged_attention(int type, int head_dim) { return paged_dispatch(type, head_dim, AttnLoad{}); }

size_t paged_attn_workspace(const ssd_ctx* ctx, int head_dim) {
    const int ctas = ctx->num_sms;
    return paged_counter_bytes(ctas) +
           (size_t)ctas * (2 + kPagedMaxWarps) * (8 * (head_dim + 4) * 4 + 64);
}

int launch_paged_attention(ssd_ctx* ctx, int type, int head_dim, const PagedAttnArgs& a,
                           cudaStream_t s, bool pdl) {
    const int64_t cap = (int64_t)a.v.pages_per_seq << a.v.page_shift;
    const int64_t most = a.window > 0 && a.window < cap ? a.window : cap;  // positions of a row
    SSD_REQ(a.n_rows * (most / kPagedGroup + 4) * a.v.n_head_kv * a.subs <= 0x7fffffff, SSD_ERR_SHAPE,
            "%d rows over %lld positions are too many for one call", a.n_rows, (long long)most);
    return paged_dispatch(type, head_dim, AttnLaunch{ctx, a, s, pdl});
}

}  // namespace ssd
