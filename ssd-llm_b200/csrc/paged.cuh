// paged.cuh — the paged KV cache's memory layout and the element access of its kernels.
//
// A pool of pages; a page holds page_size positions (a power of two, 16 or more) of every KV
// head, K and V. Which pages a sequence has, in order, is the caller's table. Inside a page the
// order is [head][16-position group], and a group (group_bytes, contiguous) is its K, then its V:
//   elements [head_dim/32 blocks][128 quads of 4 dims], in the order given by k_quad / v_quad
//   scales (Q8_0 and Q4_0 only), f16: K [16 positions][head_dim/32],
//                                     V [8 pairs of positions][head_dim/32][2]
// A group is the 16 positions of one m16n8k16 step of the attention: its K, or its V, is one bulk
// copy into shared memory, where each lane of a warp finds exactly the elements of its tensor-core
// fragments in 16-byte runs next to its neighbours' (K needs runs of dims of a position, V four
// positions of the same dims). A position's row is still made of whole quads (8, 4 or 2 bytes),
// which is what the kernel that writes rows stores per lane.
//
// Element codes: F16 / BF16 as they are; Q4_0 the format's own unsigned nibble (value nibble - 8),
// element i of a quad in bits 4i. Q8_0: sign and magnitude, two elements (X, Y) to 16 bits: |X| in
// bits 0-6, the sign of X in bit 15, |Y| in bits 8-14, the sign of Y in bit 7, so that masking with
// 0x807F leaves X, and masking the swapped bytes leaves Y, as an f16 number (a subnormal,
// q 2^-24, exact). The X, Y of a quad: dims (0, 2) and (1, 3) in K, (0, 1) and (2, 3) in V; in V
// the two halves lie in separate words, each beside the other position's of a pair.
// Value = code * the block's f16 scale.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace ssd {

constexpr int kPagedGroup = 16;  // positions of one group

__host__ __device__ constexpr bool paged_quantized(int type) {
    return type == SSD_TYPE_Q8_0 || type == SSD_TYPE_Q4_0;
}
__host__ __device__ constexpr int paged_quad_bytes(int type) {
    return type == SSD_TYPE_Q8_0 ? 4 : (type == SSD_TYPE_Q4_0 ? 2 : 8);
}
// Bytes of a group's K (or V) elements, of these with their scales, and of the group.
__host__ __device__ constexpr int paged_elem_bytes(int type, int head_dim) {
    return kPagedGroup * (head_dim / 4) * paged_quad_bytes(type);
}
__host__ __device__ constexpr int paged_half_bytes(int type, int head_dim) {
    return paged_elem_bytes(type, head_dim) +
           (paged_quantized(type) ? kPagedGroup * (head_dim / 32) * 2 : 0);
}
__host__ __device__ constexpr int paged_group_bytes(int type, int head_dim) {
    return 2 * paged_half_bytes(type, head_dim);
}

// What a kernel needs of a paged cache and of the caller's table.
struct PagedView {
    uint8_t* pool;
    const int32_t* table;  // [n_seq][pages_per_seq], page ids
    int n_pages, page_shift, n_head_kv, n_seq, pages_per_seq;
    uint32_t head_bytes;  // of one head in a page
    uint64_t page_bytes;
};

// Place of quad q (0..head_dim/4) of position t (0..15) among a group's K / V elements, in quads.
// Lane 4g + t' of a tensor-core warp owns, of every block of 32 dims,
//   of K: dims 8t'..8t'+7 (two quads) at positions g and g + 8;
//   of V: dims 4g..4g+3 (one quad) at positions 2t', 2t'+1, 2t'+8, 2t'+9.
// 8- and 4-bit types: the lane's four quads are consecutive (one read of 16 or 8 bytes); 16-bit
// types: two runs of two quads, so that each is one 16-byte read and a warp's runs are contiguous.
template <int TYPE>
__device__ __forceinline__ int k_quad(int t, int q) {
    const int b = q >> 3, lane = (t & 7) * 4 + ((q & 7) >> 1), hi = t >> 3;
    if constexpr (paged_quantized(TYPE)) return b * 128 + lane * 4 + hi * 2 + (q & 1);
    return b * 128 + hi * 64 + lane * 2 + (q & 1);
}
template <int TYPE>
__device__ __forceinline__ int v_quad(int t, int q) {
    const int b = q >> 3, lane = (q & 7) * 4 + ((t & 7) >> 1), hi = t >> 3;
    if constexpr (paged_quantized(TYPE)) return b * 128 + lane * 4 + hi * 2 + (t & 1);
    return b * 128 + hi * 64 + lane * 2 + (t & 1);
}
// Q8_0's V: the 16-bit words (dims 0, 1) and (dims 2, 3) of that quad, in 16-bit units.
__device__ __forceinline__ int v_half8(int t, int q, int i) {
    return (v_quad<SSD_TYPE_Q8_0>(t, q) & ~1) * 2 + 2 * i + (t & 1);
}
// Q8_0: sign and magnitude of X and Y in 16 bits.
__device__ __forceinline__ uint32_t pack8(int x, int y) {
    const uint32_t ax = (uint32_t)abs(x), ay = (uint32_t)abs(y);
    return ax | (x < 0 ? 0x8000u : 0u) | ay << 8 | (y < 0 ? 0x80u : 0u);
}

// Index of the scale of position t's block b among the scales of a group's K / V.
template <int HD>
__device__ __forceinline__ int paged_scale(int which, int t, int b) {
    constexpr int nb = HD / 32;
    return which ? (t >> 1) * 2 * nb + 2 * b + (t & 1) : t * nb + b;
}

// The page of (sequence, position): -1 if there is none.
__device__ __forceinline__ int paged_page(const PagedView& v, int seq, int pos) {
    const int i = pos >> v.page_shift;
    if (pos < 0 || (unsigned)seq >= (unsigned)v.n_seq || i >= v.pages_per_seq) return -1;
    const int page = v.table[(size_t)seq * v.pages_per_seq + i];
    return (unsigned)page < (unsigned)v.n_pages ? page : -1;
}
// First byte of the group that holds position `pos` of `head` in `page`.
template <int TYPE, int HD>
__device__ __forceinline__ uint8_t* paged_group(const PagedView& v, int page, int head, int pos) {
    const int in_page = (pos & ((1 << v.page_shift) - 1)) / kPagedGroup;
    return v.pool + (uint64_t)page * v.page_bytes + (size_t)head * v.head_bytes +
           (size_t)in_page * paged_group_bytes(TYPE, HD);
}

// Quad q at position t of a group's K (which = 0) or V (1): as held (the load), then its values.
struct PagedQuad {
    uint2 w;
    uint16_t d;
};
template <int TYPE, int HD>
__device__ __forceinline__ PagedQuad paged_load_quad(const uint8_t* group, int which, int t, int q) {
    const uint8_t* part = group + which * paged_half_bytes(TYPE, HD);
    const int at = which ? v_quad<TYPE>(t, q) : k_quad<TYPE>(t, q);
    const uint8_t* p = part + (size_t)at * paged_quad_bytes(TYPE);
    PagedQuad r = {};
    if constexpr (!paged_quantized(TYPE)) {
        r.w = *reinterpret_cast<const uint2*>(p);
    } else {
        r.d = reinterpret_cast<const uint16_t*>(part + paged_elem_bytes(TYPE, HD))[paged_scale<HD>(which, t, q >> 3)];
        if constexpr (TYPE == SSD_TYPE_Q4_0) {
            r.w.x = *reinterpret_cast<const uint16_t*>(p);
        } else if (which) {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(part);
            r.w = make_uint2(h[v_half8(t, q, 0)], h[v_half8(t, q, 1)]);
        } else {
            r.w.x = *reinterpret_cast<const uint32_t*>(p);
        }
    }
    return r;
}
// The four quads that lane 4g + t' owns of block b (k_quad, v_quad), in the order in which they are
// held: K: position g: quads 2t', 2t'+1, then position g + 8; V: positions 2t', 2t'+1, 2t'+8, 2t'+9.
template <int TYPE, int HD>
__device__ __forceinline__ void paged_load_lane(const uint8_t* group, int which, int b, int lane,
                                                PagedQuad (&r)[4]) {
    const uint8_t* part = group + which * paged_half_bytes(TYPE, HD);
    if constexpr (!paged_quantized(TYPE)) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint4 w = *reinterpret_cast<const uint4*>(part + (b * 2 + i) * 512 + lane * 16);
            r[2 * i].w = make_uint2(w.x, w.y);
            r[2 * i + 1].w = make_uint2(w.z, w.w);
        }
    } else {
        const uint16_t* d = reinterpret_cast<const uint16_t*>(part + paged_elem_bytes(TYPE, HD));
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (which) {
                const uint32_t p = *reinterpret_cast<const uint32_t*>(
                    d + paged_scale<HD>(1, 2 * (lane & 3) + 8 * i, b));
                r[2 * i].d = (uint16_t)p;
                r[2 * i + 1].d = (uint16_t)(p >> 16);
            } else {
                r[2 * i].d = r[2 * i + 1].d = d[paged_scale<HD>(0, (lane >> 2) + 8 * i, b)];
            }
        }
        if constexpr (TYPE == SSD_TYPE_Q4_0) {
            const uint2 w = *reinterpret_cast<const uint2*>(part + b * 256 + lane * 8);
            r[0].w.x = w.x & 0xFFFFu, r[1].w.x = w.x >> 16;
            r[2].w.x = w.y & 0xFFFFu, r[3].w.x = w.y >> 16;
        } else {
            const uint4 w = *reinterpret_cast<const uint4*>(part + b * 512 + lane * 16);
            if (which) {
                r[0].w = make_uint2(w.x & 0xFFFFu, w.y & 0xFFFFu), r[1].w = make_uint2(w.x >> 16, w.y >> 16);
                r[2].w = make_uint2(w.z & 0xFFFFu, w.w & 0xFFFFu), r[3].w = make_uint2(w.z >> 16, w.w >> 16);
            } else {
                r[0].w.x = w.x, r[1].w.x = w.y, r[2].w.x = w.z, r[3].w.x = w.w;
            }
        }
    }
}
template <int TYPE>
__device__ __forceinline__ float4 paged_quad_values(const PagedQuad& r, int which) {
    if constexpr (TYPE == SSD_TYPE_F16) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.w.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.w.y));
        return make_float4(a.x, a.y, b.x, b.y);
    } else if constexpr (TYPE == SSD_TYPE_BF16) {
        return make_float4(__uint_as_float(r.w.x << 16), __uint_as_float(r.w.x & 0xFFFF0000u),
                           __uint_as_float(r.w.y << 16), __uint_as_float(r.w.y & 0xFFFF0000u));
    } else if constexpr (TYPE == SSD_TYPE_Q8_0) {
        // X and Y of both halves as f16 numbers q 2^-24; d 2^24 takes the factor back, exactly
        const float d = __fmul_rn(f16_bits_to_f32(r.d), 16777216.0f);
        const uint32_t w = which ? r.w.x | r.w.y << 16 : r.w.x;
        const uint32_t x = w & 0x807F807Fu, y = __byte_perm(w, 0, 0x2301) & 0x807F807Fu;
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&y));
        // X: dims 0 and 1 (K) or 0 and 2 (V); Y: the other two
        return which ? make_float4(__fmul_rn(a.x, d), __fmul_rn(b.x, d), __fmul_rn(a.y, d), __fmul_rn(b.y, d))
                     : make_float4(__fmul_rn(a.x, d), __fmul_rn(a.y, d), __fmul_rn(b.x, d), __fmul_rn(b.y, d));
    } else {
        const float d = f16_bits_to_f32(r.d);
        float c[4];
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = (float)((int)((r.w.x >> (4 * i)) & 0xFu) - 8);
        return make_float4(__fmul_rn(c[0], d), __fmul_rn(c[1], d), __fmul_rn(c[2], d), __fmul_rn(c[3], d));
    }
}

// Four consecutive floats; one 16-byte load where the row allows it.
__device__ __forceinline__ float4 load4(const float* p, bool vec) {
    if (vec) return *reinterpret_cast<const float4*>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ void store4(float* p, const float4& v, bool vec) {
    if (vec) {
        *reinterpret_cast<float4*>(p) = v;
    } else {
        p[0] = v.x;
        p[1] = v.y;
        p[2] = v.z;
        p[3] = v.w;
    }
}

// ------------------------------------------------------------ host side
struct PagedAttnArgs {
    PagedView v;
    const float* q;
    float* out;
    int64_t q_stride, out_stride;
    const int32_t* len;
    const int32_t* seq;  // null: row r is sequence r
    int n_rows, n_head, window;
    int group, subs;  // query heads of a KV head, and groups of 8 of them
    float scale;
    uint8_t* work;
    int* status;  // device status word (bounded waits)
    bool q_vec, out_vec;  // rows start on 16-byte boundaries
};
size_t paged_attn_workspace(const ssd_ctx* ctx, int head_dim);
// Loads what the calls on a cache of this type and head size may launch, on the current device: with
// lazy loading the first launch of a kernel would do it, which a stream capture may not allow.
int load_paged_attention(int type, int head_dim);
int launch_paged_attention(ssd_ctx* ctx, int type, int head_dim, const PagedAttnArgs& a,
                           cudaStream_t s, bool pdl);

// Calls F::template run<TYPE, HD>() for a cache's type and head size (checked at creation).
template <typename F, int TYPE>
int paged_dispatch_dim(int head_dim, const F& f) {
    switch (head_dim) {
        case 64: return f.template run<TYPE, 64>();
        case 96: return f.template run<TYPE, 96>();
        case 128: return f.template run<TYPE, 128>();
        case 192: return f.template run<TYPE, 192>();
        default: return f.template run<TYPE, 256>();
    }
}
template <typename F>
int paged_dispatch(int type, int head_dim, const F& f) {
    switch (type) {
        case SSD_TYPE_F16: return paged_dispatch_dim<F, SSD_TYPE_F16>(head_dim, f);
        case SSD_TYPE_BF16: return paged_dispatch_dim<F, SSD_TYPE_BF16>(head_dim, f);
        case SSD_TYPE_Q8_0: return paged_dispatch_dim<F, SSD_TYPE_Q8_0>(head_dim, f);
        default: return paged_dispatch_dim<F, SSD_TYPE_Q4_0>(head_dim, f);
    }
}

}  // namespace ssd
