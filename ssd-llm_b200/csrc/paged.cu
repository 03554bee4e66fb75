// paged.cu — the paged KV cache: pages, the fused write of new rows (per-head RMSNorm of queries
// and keys, RoPE, rounding to the cache's type) and the read-back of its values.
//
// The reference manages pages on the CPU (src/inference/paged_attention.rs); here the pages live
// in HBM and the caller keeps the tables.
#include <new>
#include <type_traits>

#include "paged.cuh"

namespace ssd {

struct PagedAppendArgs {
    PagedView v;
    const float *q, *k, *x;  // x: the V rows
    int64_t q_stride, k_stride, x_stride;
    int n_head, n_rows;
    int q_items, k_items;                     // warps of a row for the queries, and for the keys
    // CTAs of all rows' values (the first of the grid: theirs is the longest work), of 16 rows'
    uint32_t value_ctas, head_ctas;
    const float *q_norm, *k_norm;
    float eps;
    const float2* rope;
    int rope_dim, rope_positions, rope_halves;
    const int32_t* pos;
    const int32_t* seq;
    float* q_out;
    int64_t q_out_stride;
    int* status;
    bool vec;  // every row, weight and table row starts on a 16-byte boundary
};

// Codes of four values of a block whose scale is d: ssd_quantize's rules.
template <int TYPE>
__device__ __forceinline__ void paged_codes(const float (&v)[4], float d, int (&c)[4]) {
    const float id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++)
        c[i] = TYPE == SSD_TYPE_Q8_0
                   ? min(127, max(-127, (int)roundf(__fmul_rn(v[i], id))))
                   : min(15, max(0, (int)floorf(__fadd_rn(__fmul_rn(v[i], id), 8.5f))));
}

// Stores quad `qi` of a row at position t of the group. The 8 lanes of a 32-value block (aligned
// in the warp) hold its 8 quads, so the block's scale is a reduction over 8 lanes. The rules are
// ssd_quantize's (every operation rounded to nearest, ties of the 4-bit extreme to the lowest
// index), so a row written here and one quantized there have the same codes. All lanes of the
// warp call it (in: whether this lane has a quad).
template <int TYPE, int HD>
__device__ __forceinline__ void paged_store_quad(uint8_t* group, int which, int t, int qi,
                                                 const float4& x, bool in) {
    uint8_t* part = group + which * paged_half_bytes(TYPE, HD);
    const int at = which ? v_quad<TYPE>(t, qi) : k_quad<TYPE>(t, qi);
    uint8_t* p = part + (size_t)at * paged_quad_bytes(TYPE);
    if constexpr (TYPE == SSD_TYPE_F16) {
        if (!in) return;
        const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                                  *reinterpret_cast<const uint32_t*>(&b));
    } else if constexpr (TYPE == SSD_TYPE_BF16) {
        if (!in) return;
        const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                                  *reinterpret_cast<const uint32_t*>(&b));
    } else {
        const float v[4] = {x.x, x.y, x.z, x.w};
        float am = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) am = fmaxf(am, fabsf(v[i]));
        float top = am;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float d;
        if constexpr (TYPE == SSD_TYPE_Q8_0) {
            d = __fdiv_rn(top, 127.0f);
        } else {
            float m = 0.0f;  // this lane's first value of the block's largest magnitude
#pragma unroll
            for (int i = 3; i >= 0; i--) m = fabsf(v[i]) == top ? v[i] : m;
            const int lane = threadIdx.x & 31;
            const uint32_t has = __ballot_sync(0xffffffffu, am == top) & (0xFFu << (lane & 24));
            m = __shfl_sync(0xffffffffu, m, has ? __ffs((int)has) - 1 : lane);
            d = __fdiv_rn(m, -8.0f);
        }
        if (!in) return;
        int c[4];
        paged_codes<TYPE>(v, d, c);
        if constexpr (TYPE == SSD_TYPE_Q4_0) {
            *reinterpret_cast<uint16_t*>(p) = (uint16_t)(c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12);
        } else if (which) {
            uint16_t* h = reinterpret_cast<uint16_t*>(part);
            h[v_half8(t, qi, 0)] = (uint16_t)pack8(c[0], c[1]);
            h[v_half8(t, qi, 1)] = (uint16_t)pack8(c[2], c[3]);
        } else {
            *reinterpret_cast<uint32_t*>(p) = pack8(c[0], c[2]) | pack8(c[1], c[3]) << 16;
        }
        if ((qi & 7) == 0)
            reinterpret_cast<uint16_t*>(
                part + paged_elem_bytes(TYPE, HD))[paged_scale<HD>(which, t, qi >> 3)] =
                __half_as_ushort(__float2half_rn(d));
    }
}

// Up to 16 rows from r0 on: how many there are, and whether they are consecutive positions of one
// sequence that its row of the page table reaches (of which the first is then `pos` of `seq`): what
// lies beyond goes row by row, so that no loop over a run's positions comes near INT_MAX. All lanes
// of the warp call it.
struct PagedRun {
    int n, seq, pos;
    bool run;
};
__device__ __forceinline__ PagedRun paged_run(const PagedView& v, const int32_t* pos, const int32_t* seq,
                                              int r0, int n_rows) {
    const int lane = threadIdx.x & 31;
    PagedRun u;
    u.n = min(16, n_rows - r0);
    const int i = min(lane, u.n - 1);
    const int p = pos[r0 + i], q = seq ? seq[r0 + i] : r0 + i;
    u.pos = __shfl_sync(0xffffffffu, p, 0);
    u.seq = __shfl_sync(0xffffffffu, q, 0);
    const int last = (v.pages_per_seq << v.page_shift) - u.n;  // at most 2^31 - 1 positions
    u.run = __all_sync(0xffffffffu, q == u.seq && (uint32_t)p - (uint32_t)u.pos == (uint32_t)i) &&
            u.pos >= 0 && u.pos <= last;
    return u;
}

// V of 16 consecutive positions (rows r0 .. r0 + n, the first at `pos`) of one head, in the order
// in which it is held: lane 4 g + t takes dims 4 g .. 4 g + 3 of every block at positions 2 t,
// 2 t + 1, 2 t + 8, 2 t + 9 of a group, so that a warp reads whole lines of the rows and writes
// whole lines of the cache (a row at a time, a lane's two to eight bytes lie 64 bytes from the next
// lane's).
template <int TYPE, int HD, bool VEC>
__device__ __forceinline__ void paged_store_v(const PagedView& v, const float* src, int64_t stride,
                                              int head, int seq, int pos, int n) {
    constexpr int NB = HD / 32;
    const int lane = threadIdx.x & 31, g = lane >> 2, t2 = 2 * (lane & 3);
    src += (size_t)head * HD + 4 * g;
    for (int p0 = pos & ~15; p0 < pos + n; p0 += 16) {  // one group, or two
        const int page = paged_page(v, seq, p0);
        uint8_t* part = paged_group<TYPE, HD>(v, max(page, 0), head, p0) + paged_half_bytes(TYPE, HD);
        const bool all = p0 >= pos && p0 + 16 <= pos + n;
        constexpr int AT = NB % 2 == 0 ? 2 : 3;  // blocks in flight
        float4 y[AT][4];
#pragma unroll AT
        for (int b = 0; b < NB; b++) {
            if (b % AT == 0) {  // the rows' loads, before the page is known
#pragma unroll
                for (int i = 0; i < AT; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int r = p0 + t2 + (j & 1) + 8 * (j >> 1) - pos;
                        y[i][j] = r >= 0 && r < n ? load4(src + r * stride + 32 * (b + i), VEC)
                                                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                if (page < 0) break;  // the rows' own look-up reports it
            }
            float4(&x)[4] = y[b % AT];
            if constexpr (!paged_quantized(TYPE)) {
                uint2 w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (TYPE == SSD_TYPE_F16) {
                        const __half2 lo = __floats2half2_rn(x[j].x, x[j].y), hi = __floats2half2_rn(x[j].z, x[j].w);
                        w[j] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
                    } else {
                        const __nv_bfloat162 lo = __floats2bfloat162_rn(x[j].x, x[j].y), hi = __floats2bfloat162_rn(x[j].z, x[j].w);
                        w[j] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    uint8_t* o = part + (b * 2 + i) * 512 + lane * 16;
                    if (all) {
                        *reinterpret_cast<uint4*>(o) = make_uint4(w[2 * i].x, w[2 * i].y, w[2 * i + 1].x, w[2 * i + 1].y);
                    } else {
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const int r = p0 + t2 + k + 8 * i - pos;
                            if (r >= 0 && r < n) *reinterpret_cast<uint2*>(o + 8 * k) = w[2 * i + k];
                        }
                    }
                }
            } else {
                uint32_t h[4][2];  // 16-bit words of the lane's quads (Q4_0: one)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float f[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
                    float am = fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3])));
                    float top = am;
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    float d;
                    if constexpr (TYPE == SSD_TYPE_Q8_0) {
                        d = __fdiv_rn(top, 127.0f);
                    } else {
                        float m = 0.0f;
#pragma unroll
                        for (int k = 3; k >= 0; k--) m = fabsf(f[k]) == top ? f[k] : m;
                        const uint32_t has = __ballot_sync(0xffffffffu, am == top) & (0x11111111u << (lane & 3));
                        m = __shfl_sync(0xffffffffu, m, has ? __ffs((int)has) - 1 : lane);
                        d = __fdiv_rn(m, -8.0f);
                    }
                    int c[4];
                    paged_codes<TYPE>(f, d, c);
                    if constexpr (TYPE == SSD_TYPE_Q4_0) {
                        h[j][0] = (uint32_t)(c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12);
                    } else {
                        h[j][0] = pack8(c[0], c[1]);
                        h[j][1] = pack8(c[2], c[3]);
                    }
                    const int t = t2 + (j & 1) + 8 * (j >> 1), r = p0 + t - pos;
                    if (g == 0 && r >= 0 && r < n)
                        reinterpret_cast<uint16_t*>(part + paged_elem_bytes(TYPE, HD))[paged_scale<HD>(1, t, b)] =
                            __half_as_ushort(__float2half_rn(d));
                }
                constexpr int HW = TYPE == SSD_TYPE_Q8_0 ? 2 : 1;
                uint8_t* o = part + b * (256 * HW) + lane * (8 * HW);
                if (all) {
                    if constexpr (HW == 2)
                        *reinterpret_cast<uint4*>(o) = make_uint4(h[0][0] | h[1][0] << 16, h[0][1] | h[1][1] << 16,
                                                                  h[2][0] | h[3][0] << 16, h[2][1] | h[3][1] << 16);
                    else
                        *reinterpret_cast<uint2*>(o) = make_uint2(h[0][0] | h[1][0] << 16, h[2][0] | h[3][0] << 16);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int r = p0 + t2 + (j & 1) + 8 * (j >> 1) - pos;
                        if (r < 0 || r >= n) continue;
#pragma unroll
                        for (int k = 0; k < HW; k++)
                            reinterpret_cast<uint16_t*>(o)[(j >> 1) * 2 * HW + 2 * k + (j & 1)] = (uint16_t)h[j][k];
                    }
                }
            }
        }
    }
}

// Queries and keys: one warp per (row, kHeads heads of one kind). Values: one warp per (16 rows,
// head) where the rows are consecutive positions, else per row.
//   queries, keys: n_i = x_i (w_i / sqrt(mean x^2 + eps)) where there is a norm weight, then the
//   pair rotation (a, b) -> (a c - b s, a s + b c), pairs (2i, 2i+1) or (i, i + rope_dim/2);
//   values: as they are.
// Of queries and keys a lane holds quads i and i + L of a head (4 dims each, L half the head's quads), so that the pairs
// of a rotation of the whole head lie in one lane, and 32 / L heads side by side; heads of 96, whose
// half is no whole number of the formats' blocks, one head and quads i and i + 32.
// Bound by HBM: each input and output is moved once. The heads' rows are loaded before the page is
// looked up, and kHeads heads share the look-up and the norm's and the rotation's loads, so that
// kilobytes a warp are in flight. 4096 rows of 64 / 8 heads of 128, BF16: 58.6 us, 5.4 TB/s (one head
// a warp, each behind its own look-up: 85).
constexpr int kHeads = 4;
template <int HD>
struct AppendCfg {
    static constexpr int NQ = HD / 4;
    static constexpr int L = HD == 96 ? 32 : NQ / 2;     // lanes of a head
    static constexpr int SIDE = 32 / L;                  // heads side by side
    static constexpr int STEPS = (kHeads + SIDE - 1) / SIDE;
    static constexpr int HEADS = STEPS * SIDE;           // heads of a warp
    static constexpr int NC = HD == 96 ? 1 : 2;          // quads of a lane and step
};
template <int TYPE, int HD, bool VEC>
__global__ void __launch_bounds__(256, HD <= 128 ? 4 : 3) k_paged_append(const PagedAppendArgs a) {
    using C = AppendCfg<HD>;
    constexpr int NQ = C::NQ, NC = C::NC, ST = C::STEPS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    if (blockIdx.x < a.value_ctas) {  // ---- values: 16 rows, 8 heads
        const uint32_t block = blockIdx.x / a.head_ctas;
        const int r0 = (int)block * 16, hv = (int)(blockIdx.x - block * a.head_ctas) * 8;
        const PagedRun u = paged_run(a.v, a.pos, a.seq, r0, a.n_rows);
        if (u.run) {
            if (hv + warp < a.v.n_head_kv)
                paged_store_v<TYPE, HD, VEC>(a.v, a.x + (int64_t)r0 * a.x_stride, a.x_stride, hv + warp,
                                             u.seq, u.pos, a.rope ? min(u.n, a.rope_positions - u.pos) : u.n);
            return;
        }
        for (int r = warp; r < u.n; r += 8) {  // rows of their own
            const int row = r0 + r, pos = a.pos[row];
            const int page = paged_page(a.v, a.seq ? a.seq[row] : row, pos);
            if (page < 0 || (a.rope && pos >= a.rope_positions)) continue;
            uint8_t* group = paged_group<TYPE, HD>(a.v, page, hv, pos);
            const float* src = a.x + (int64_t)row * a.x_stride + (size_t)hv * HD;
            const int nh = min(8, a.v.n_head_kv - hv);
#pragma unroll 4
            for (int h = 0; h < nh; h++)
#pragma unroll
                for (int c = 0; c < (NQ + 31) / 32; c++) {
                    const int qi = lane + 32 * c;
                    const float4 x = qi < NQ ? load4(src + h * HD + 4 * qi, VEC)
                                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    paged_store_quad<TYPE, HD>(group + (size_t)h * a.v.head_bytes, 1, pos & 15, qi, x, qi < NQ);
                }
        }
        return;
    }
    // ---- queries and keys
    const uint32_t items = (uint32_t)(a.q_items + a.k_items), i = (blockIdx.x - a.value_ctas) * 8 + warp;
    const int row = (int)(i / items), hs = (int)(i - (uint32_t)row * items);
    if (row >= a.n_rows) return;
    const int kind = hs < a.q_items ? 0 : 1;
    const int h0 = (kind == 0 ? hs : hs - a.q_items) * C::HEADS;
    const int nh = min(C::HEADS, (kind == 0 ? a.n_head : a.v.n_head_kv) - h0);
    const float* src = kind == 0 ? a.q + (int64_t)row * a.q_stride : a.k + (int64_t)row * a.k_stride;
    src += (size_t)h0 * HD;
    const int side = lane / C::L, li = lane % C::L;      // lanes beyond the heads: side >= SIDE
    auto quad = [&](int c) { return li + c * C::L; };    // quad of the head
    auto head = [&](int st) { return st * C::SIDE + side; };
    auto in = [&](int st, int c) { return side < C::SIDE && head(st) < nh && quad(c) < NQ; };
    float4 x[ST][NC];
#pragma unroll
    for (int st = 0; st < ST; st++)
#pragma unroll
        for (int c = 0; c < NC; c++)
            x[st][c] = in(st, c) ? load4(src + head(st) * HD + 4 * quad(c), VEC)
                                 : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int pos = a.pos[row], page = paged_page(a.v, a.seq ? a.seq[row] : row, pos);
    const bool ok = page >= 0 && (!a.rope || pos < a.rope_positions);
    float* q_out = kind == 0 ? a.q_out + (int64_t)row * a.q_out_stride + (size_t)h0 * HD : nullptr;
    if (!ok) {  // padding (pos < 0) or a position without a page: nothing is kept
        if (pos >= 0 && hs == 0 && lane == 0) atomicCAS(a.status, SSD_OK, SSD_ERR_SHAPE);
        if (kind == 0)
            for (int i = lane; i < nh * NQ; i += 32)
                store4(q_out + 4 * i, make_float4(0.0f, 0.0f, 0.0f, 0.0f), VEC);
        return;
    }
    const float* w = kind == 0 ? a.q_norm : a.k_norm;
    if (w) {
        float ss[ST], mine = 0.0f;
#pragma unroll
        for (int st = 0; st < ST; st++) {
            ss[st] = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const float4& y = x[st][c];
                ss[st] = fmaf(y.x, y.x, fmaf(y.y, y.y, fmaf(y.z, y.z, fmaf(y.w, y.w, ss[st]))));
            }
        }
        // the sum over the lanes of a head (a power of two of them, or 24, whose third 8 follow)
        constexpr int P2 = C::L == 24 ? 8 : C::L;
#pragma unroll
        for (int o = P2 / 2; o > 0; o >>= 1)
#pragma unroll
            for (int st = 0; st < ST; st++) ss[st] += __shfl_xor_sync(0xffffffffu, ss[st], o);
        if constexpr (C::L == 24) {
#pragma unroll
            for (int st = 0; st < ST; st++)
                ss[st] = (__shfl_sync(0xffffffffu, ss[st], 0) + __shfl_sync(0xffffffffu, ss[st], 8)) +
                         __shfl_sync(0xffffffffu, ss[st], 16);
        }
        // 1 / sqrt once for each head: lane st of a head's lanes does step st's
#pragma unroll
        for (int st = 0; st < ST; st++) mine = (li % ST) == st ? ss[st] : mine;
        mine = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(mine, (float)HD), a.eps)));
        float4 g[NC];
#pragma unroll
        for (int c = 0; c < NC; c++)
            g[c] = quad(c) < NQ ? load4(w + 4 * quad(c), VEC) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int st = 0; st < ST; st++) {
            const float inv = __shfl_sync(0xffffffffu, mine, (min(side, C::SIDE - 1) * C::L + st));
#pragma unroll
            for (int c = 0; c < NC; c++) {
                x[st][c].x = __fmul_rn(x[st][c].x, __fmul_rn(inv, g[c].x));
                x[st][c].y = __fmul_rn(x[st][c].y, __fmul_rn(inv, g[c].y));
                x[st][c].z = __fmul_rn(x[st][c].z, __fmul_rn(inv, g[c].z));
                x[st][c].w = __fmul_rn(x[st][c].w, __fmul_rn(inv, g[c].w));
            }
        }
    }
    if (a.rope) {
        const float* cs = reinterpret_cast<const float*>(a.rope + (size_t)pos * (a.rope_dim / 2));
        const int nr = a.rope_dim / 4;  // quads that rotate
        if (!a.rope_halves) {
#pragma unroll
            for (int c = 0; c < NC; c++) {
                if (quad(c) >= nr) continue;
                const float4 t = load4(cs + 4 * quad(c), VEC);
#pragma unroll
                for (int st = 0; st < ST; st++) {
                    const float4 y = x[st][c];
                    x[st][c].x = __fsub_rn(__fmul_rn(y.x, t.x), __fmul_rn(y.y, t.y));
                    x[st][c].y = __fadd_rn(__fmul_rn(y.x, t.y), __fmul_rn(y.y, t.x));
                    x[st][c].z = __fsub_rn(__fmul_rn(y.z, t.z), __fmul_rn(y.w, t.w));
                    x[st][c].w = __fadd_rn(__fmul_rn(y.z, t.w), __fmul_rn(y.w, t.z));
                }
            }
        } else if (NC == 2 && a.rope_dim == HD) {  // the pair's halves are the lane's two quads
            const int qi = min(quad(0), NQ / 2 - 1);
            const float4 t0 = load4(cs + 8 * qi, VEC), t1 = load4(cs + 8 * qi + 4, VEC);
#pragma unroll
            for (int st = 0; st < ST; st++) {
                const float4 y = x[st][0], z = x[st][NC - 1];
                x[st][0].x = __fsub_rn(__fmul_rn(y.x, t0.x), __fmul_rn(z.x, t0.y));
                x[st][0].y = __fsub_rn(__fmul_rn(y.y, t0.z), __fmul_rn(z.y, t0.w));
                x[st][0].z = __fsub_rn(__fmul_rn(y.z, t1.x), __fmul_rn(z.z, t1.y));
                x[st][0].w = __fsub_rn(__fmul_rn(y.w, t1.z), __fmul_rn(z.w, t1.w));
                x[st][NC - 1].x = __fadd_rn(__fmul_rn(y.x, t0.y), __fmul_rn(z.x, t0.x));
                x[st][NC - 1].y = __fadd_rn(__fmul_rn(y.y, t0.w), __fmul_rn(z.y, t0.z));
                x[st][NC - 1].z = __fadd_rn(__fmul_rn(y.z, t1.y), __fmul_rn(z.z, t1.x));
                x[st][NC - 1].w = __fadd_rn(__fmul_rn(y.w, t1.w), __fmul_rn(z.w, t1.z));
            }
        } else {  // a quad's partner is nr / 2 quads away, in another lane
#pragma unroll
            for (int st = 0; st < ST; st++) {
                float4 o[NC];
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const int qi = quad(c), pq = max(0, qi < nr / 2 ? qi + nr / 2 : qi - nr / 2);
                    const int from = min(side, C::SIDE - 1) * C::L + pq % C::L;
                    o[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int e = 0; e < NC; e++) {
                        const float4 y = make_float4(__shfl_sync(0xffffffffu, x[st][e].x, from),
                                                     __shfl_sync(0xffffffffu, x[st][e].y, from),
                                                     __shfl_sync(0xffffffffu, x[st][e].z, from),
                                                     __shfl_sync(0xffffffffu, x[st][e].w, from));
                        if (pq / C::L == e) o[c] = y;
                    }
                }
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const int qi = quad(c);
                    if (qi >= nr) continue;
                    const bool first = qi < nr / 2;
                    const int i = first ? qi : qi - nr / 2;
                    const float4 t0 = load4(cs + 8 * i, VEC), t1 = load4(cs + 8 * i + 4, VEC);
                    const float4 y = x[st][c];
                    if (first) {
                        x[st][c].x = __fsub_rn(__fmul_rn(y.x, t0.x), __fmul_rn(o[c].x, t0.y));
                        x[st][c].y = __fsub_rn(__fmul_rn(y.y, t0.z), __fmul_rn(o[c].y, t0.w));
                        x[st][c].z = __fsub_rn(__fmul_rn(y.z, t1.x), __fmul_rn(o[c].z, t1.y));
                        x[st][c].w = __fsub_rn(__fmul_rn(y.w, t1.z), __fmul_rn(o[c].w, t1.w));
                    } else {
                        x[st][c].x = __fadd_rn(__fmul_rn(o[c].x, t0.y), __fmul_rn(y.x, t0.x));
                        x[st][c].y = __fadd_rn(__fmul_rn(o[c].y, t0.w), __fmul_rn(y.y, t0.z));
                        x[st][c].z = __fadd_rn(__fmul_rn(o[c].z, t1.y), __fmul_rn(y.z, t1.x));
                        x[st][c].w = __fadd_rn(__fmul_rn(o[c].w, t1.w), __fmul_rn(y.w, t1.z));
                    }
                }
            }
        }
    }
    uint8_t* group0 = paged_group<TYPE, HD>(a.v, page, kind ? h0 : 0, pos);
#pragma unroll
    for (int st = 0; st < ST; st++) {
        if (st * C::SIDE >= nh) break;
        uint8_t* group = group0 + (size_t)min(head(st), nh - 1) * a.v.head_bytes;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            if (kind == 0) {
                if (in(st, c)) store4(q_out + head(st) * HD + 4 * quad(c), x[st][c], VEC);
            } else {
                paged_store_quad<TYPE, HD>(group, 0, pos & 15, quad(c), x[st][c], in(st, c));
            }
        }
    }
}

struct PagedReadArgs {
    PagedView v;
    int n_rows, out_type;
    const int32_t* pos;
    const int32_t* seq;
    uint8_t *k, *x;  // x: the V rows
    int64_t k_stride, x_stride;  // elements
    bool vec;                    // rows start on the boundary of a quad
};

// CTA: 16 rows, 8 KV heads. Where the rows are consecutive positions, one warp per head: it reads
// whole lines of the one or two groups that hold them, each lane its 16 bytes (of K: 8 dims of two
// positions, of V: 4 dims of four), and writes whole sectors of the rows. Else one warp per row,
// the loads of four heads in flight. 32768 positions of 8 heads of 128, Q8_0 to F16: 47 us, 4.4 TB/s
// read and written, two thirds of a copy's rate (every row on its own 57; its keys and its values of
// each head on their own 94). Latency bounds it: 31 % of the warps an SM could hold are there (76 to
// 108 registers), and they issue in 35 % of the cycles.
template <int OUT, bool VEC>
__device__ __forceinline__ void paged_emit(void* out, int64_t at, const float4& v) {
    if constexpr (OUT == SSD_TYPE_F32) {
        store4(reinterpret_cast<float*>(out) + at, v, VEC);
    } else {
        uint32_t lo, hi;
        if constexpr (OUT == SSD_TYPE_F16) {
            const __half2 p = __floats2half2_rn(v.x, v.y), q = __floats2half2_rn(v.z, v.w);
            lo = *reinterpret_cast<const uint32_t*>(&p);
            hi = *reinterpret_cast<const uint32_t*>(&q);
        } else {
            const __nv_bfloat162 p = __floats2bfloat162_rn(v.x, v.y), q = __floats2bfloat162_rn(v.z, v.w);
            lo = *reinterpret_cast<const uint32_t*>(&p);
            hi = *reinterpret_cast<const uint32_t*>(&q);
        }
        uint16_t* o = reinterpret_cast<uint16_t*>(out) + at;
        if constexpr (VEC) {
            *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
        } else {
            o[0] = (uint16_t)lo, o[1] = (uint16_t)(lo >> 16);
            o[2] = (uint16_t)hi, o[3] = (uint16_t)(hi >> 16);
        }
    }
}
template <int TYPE, int HD, int OUT, bool VEC>
__device__ __forceinline__ void paged_read_run(const PagedReadArgs& a, int r0, int head, const PagedRun& u) {
    constexpr int NB = HD / 32;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t ka = (int64_t)r0 * a.k_stride + (int64_t)head * HD + 8 * t;
    const int64_t xa = (int64_t)r0 * a.x_stride + (int64_t)head * HD + 4 * g;
    for (int p0 = u.pos & ~15; p0 < u.pos + u.n; p0 += 16) {
        const int page = paged_page(a.v, u.seq, p0);
        const uint8_t* group = paged_group<TYPE, HD>(a.v, max(page, 0), head, p0);
#pragma unroll 4
        for (int b = 0; b < NB; b++) {
            PagedQuad k[4], v[4];
            if (page >= 0) {
                paged_load_lane<TYPE, HD>(group, 0, b, lane, k);
                paged_load_lane<TYPE, HD>(group, 1, b, lane, v);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                const int rk = p0 + g + 8 * (j >> 1) - u.pos, rv = p0 + 2 * t + (j & 1) + 8 * (j >> 1) - u.pos;
                if (rk >= 0 && rk < u.n)
                    paged_emit<OUT, VEC>(a.k, ka + rk * a.k_stride + 32 * b + 4 * (j & 1),
                                         page >= 0 ? paged_quad_values<TYPE>(k[j], 0) : zero);
                if (rv >= 0 && rv < u.n)
                    paged_emit<OUT, VEC>(a.x, xa + rv * a.x_stride + 32 * b,
                                         page >= 0 ? paged_quad_values<TYPE>(v[j], 1) : zero);
            }
        }
    }
}
template <int TYPE, int HD, int OUT, bool VEC>
__device__ __forceinline__ void paged_read_row(const PagedReadArgs& a, int row, int h0, int nh) {
    constexpr int NQ = HD / 4, NC = (NQ + 31) / 32;
    const int lane = threadIdx.x & 31;
    const int pos = a.pos[row], page = paged_page(a.v, a.seq ? a.seq[row] : row, pos);
    const uint8_t* group = paged_group<TYPE, HD>(a.v, max(page, 0), h0, max(pos, 0));
    const int t = pos & 15;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int qi = lane + 32 * c;
        if (qi >= NQ) break;
        const int64_t ka = (int64_t)row * a.k_stride + (int64_t)h0 * HD + 4 * qi;
        const int64_t xa = (int64_t)row * a.x_stride + (int64_t)h0 * HD + 4 * qi;
        for (int j0 = 0; j0 < nh; j0 += kHeads) {
            PagedQuad r[kHeads][2];
#pragma unroll
            for (int j = 0; j < kHeads; j++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    if (page >= 0 && j0 + j < nh)
                        r[j][i] = paged_load_quad<TYPE, HD>(group + (size_t)(j0 + j) * a.v.head_bytes, i, t, qi);
#pragma unroll
            for (int j = 0; j < kHeads; j++) {
                if (j0 + j >= nh) break;
                const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                paged_emit<OUT, VEC>(a.k, ka + (j0 + j) * HD,
                                     page >= 0 ? paged_quad_values<TYPE>(r[j][0], 0) : zero);
                paged_emit<OUT, VEC>(a.x, xa + (j0 + j) * HD,
                                     page >= 0 ? paged_quad_values<TYPE>(r[j][1], 1) : zero);
            }
        }
    }
}
template <int TYPE, int HD, bool VEC>
__global__ void __launch_bounds__(256) k_paged_read(const PagedReadArgs a) {
    const int warp = threadIdx.x >> 5, r0 = blockIdx.x * 16, h0 = blockIdx.y * 8;
    const int nh = min(8, a.v.n_head_kv - h0);
    pdl_wait();
    const PagedRun u = paged_run(a.v, a.pos, a.seq, r0, a.n_rows);
    auto all = [&](auto out) {
        constexpr int OUT = decltype(out)::value;
        if (!u.run) {
            for (int r = warp; r < u.n; r += 8) paged_read_row<TYPE, HD, OUT, VEC>(a, r0 + r, h0, nh);
        } else if (warp < nh) {
            paged_read_run<TYPE, HD, OUT, VEC>(a, r0, h0 + warp, u);
        }
    };
    if (a.out_type == SSD_TYPE_F16)
        all(std::integral_constant<int, SSD_TYPE_F16>());
    else if (a.out_type == SSD_TYPE_BF16)
        all(std::integral_constant<int, SSD_TYPE_BF16>());
    else
        all(std::integral_constant<int, SSD_TYPE_F32>());
}

__global__ void k_paged_rope_table(float2* t, int rope_dim, float theta) {
    const int pos = blockIdx.x, half = rope_dim / 2;
    for (int i = threadIdx.x; i < half; i += blockDim.x)
        t[(size_t)pos * half + i] = rope_cs(i, rope_dim, theta, pos);
}

static int paged_view(const ssd_kv_cache* kv, const int32_t* table, int n_seq, int pages_per_seq,
                      PagedView* v) {
    SSD_REQ(kv && table, SSD_ERR_ARG, "null pointer");
    SSD_REQ(kv->page_size > 0, SSD_ERR_STATE, "not a paged cache (ssd_kv_create_paged makes one)");
    SSD_REQ(n_seq > 0 && pages_per_seq > 0, SSD_ERR_ARG, "empty page table (%d x %d)", n_seq,
            pages_per_seq);
    SSD_REQ((int64_t)pages_per_seq * kv->page_size <= 0x7fffffff, SSD_ERR_SHAPE,
            "%d pages of %d positions exceed 2^31 - 1 positions", pages_per_seq, kv->page_size);
    v->pool = (uint8_t*)kv->base;
    v->table = table;
    v->n_pages = kv->n_pages;
    v->page_shift = __builtin_ctz(kv->page_size);
    v->n_head_kv = kv->n_head_kv;
    v->n_seq = n_seq;
    v->pages_per_seq = pages_per_seq;
    v->head_bytes = (uint32_t)(kv->page_size / kPagedGroup *
                               paged_group_bytes(kv->paged_type, kv->head_dim));
    v->page_bytes = (uint64_t)v->head_bytes * kv->n_head_kv;
    return SSD_OK;
}

static bool aligned(const void* p, int64_t stride, int elem, int to) {
    return ((uintptr_t)p % to) == 0 && (stride * elem) % to == 0;
}

struct AppendLaunch {
    const PagedAppendArgs& a;
    cudaStream_t s;
    bool pdl;
    template <int TYPE, int HD>
    int run() const {
        constexpr int n = AppendCfg<HD>::HEADS;
        PagedAppendArgs b = a;
        b.q_items = (a.n_head + n - 1) / n;
        b.k_items = (a.v.n_head_kv + n - 1) / n;
        b.head_ctas = (uint32_t)((a.v.n_head_kv + 7) / 8);
        const int64_t value_ctas = ((int64_t)a.n_rows + 15) / 16 * b.head_ctas;
        const int64_t ctas = value_ctas + ((int64_t)a.n_rows * (b.q_items + b.k_items) + 7) / 8;
        SSD_REQ(ctas <= 0x0fffffff, SSD_ERR_SHAPE, "%d rows of %d heads are too many", a.n_rows, a.n_head);
        b.value_ctas = (uint32_t)value_ctas;
        SSD_CK(launch_pdl(a.vec ? k_paged_append<TYPE, HD, true> : k_paged_append<TYPE, HD, false>,
                          dim3((unsigned)ctas), dim3(256), 0, s, pdl, b));
        return SSD_OK;
    }
};
struct ReadLaunch {
    const PagedReadArgs& a;
    cudaStream_t s;
    bool pdl;
    template <int TYPE, int HD>
    int run() const {
        SSD_CK(launch_pdl(a.vec ? k_paged_read<TYPE, HD, true> : k_paged_read<TYPE, HD, false>,
                          dim3((unsigned)((a.n_rows + 15) / 16), (unsigned)((a.v.n_head_kv + 7) / 8)),
                          dim3(256), 0, s, pdl, a));
        return SSD_OK;
    }
};

struct CacheLoad {
    template <int TYPE, int HD>
    int run() const {
        cudaFuncAttributes at;
        SSD_CK(cudaFuncGetAttributes(&at, k_paged_append<TYPE, HD, true>));
        SSD_CK(cudaFuncGetAttributes(&at, k_paged_append<TYPE, HD, false>));
        SSD_CK(cudaFuncGetAttributes(&at, k_paged_read<TYPE, HD, true>));
        SSD_CK(cudaFuncGetAttributes(&at, k_paged_read<TYPE, HD, false>));
        return load_paged_attention(TYPE, HD);
    }
};

}  // namespace ssd

using namespace ssd;

extern "C" int ssd_kv_create_paged(ssd_ctx* ctx, int n_pages, int page_size, int n_head_kv,
                                   int head_dim, int ggml_type, ssd_kv_cache** out) {
    SSD_TRY(check_ctx(ctx));
    SSD_REQ(out && n_pages > 0 && n_head_kv > 0, SSD_ERR_ARG, "bad arguments");
    SSD_REQ(ggml_type == SSD_TYPE_F16 || ggml_type == SSD_TYPE_BF16 || paged_quantized(ggml_type),
            SSD_ERR_TYPE, "paged cache type %d not supported (F16, BF16, Q8_0, Q4_0)", ggml_type);
    SSD_REQ(head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 192 || head_dim == 256,
            SSD_ERR_SHAPE, "head_dim %d not supported (64, 96, 128, 192, 256)", head_dim);
    SSD_REQ(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
            SSD_ERR_SHAPE, "page_size %d must be a power of two from 16 to 4096", page_size);
    SSD_REQ(n_head_kv <= 32767, SSD_ERR_SHAPE, "n_head_kv %d exceeds 32767", n_head_kv);
    const uint64_t head = (uint64_t)(page_size / kPagedGroup) * paged_group_bytes(ggml_type, head_dim);
    const uint64_t total = (uint64_t)n_pages * n_head_kv * head;
    SSD_REQ((double)n_pages * n_head_kv * (double)head < 1e15, SSD_ERR_NOMEM,
            "paged KV cache of %d pages is too large", n_pages);
    SSD_TRY(paged_dispatch(ggml_type, head_dim, CacheLoad{}));
    void* p = nullptr;
    if (cudaMalloc(&p, total) != cudaSuccess) {
        cudaGetLastError();
        set_error("paged KV cache allocation of %llu bytes failed", (unsigned long long)total);
        return SSD_ERR_NOMEM;
    }
    if (zero_device(ctx, p, total) != SSD_OK) {
        cudaFree(p);
        return SSD_ERR_CUDA;
    }
    ssd_kv_cache* kv = new (std::nothrow) ssd_kv_cache();
    if (!kv) {
        cudaFree(p);
        set_error("out of host memory");
        return SSD_ERR_NOMEM;
    }
    kv->ctx = ctx;
    kv->n_head_kv = n_head_kv;
    kv->head_dim = head_dim;
    kv->kv_dim = n_head_kv * head_dim;
    kv->n_pages = n_pages;
    kv->page_size = page_size;
    kv->paged_type = ggml_type;
    kv->base = p;
    *out = kv;
    return SSD_OK;
}

extern "C" int ssd_rope_table(ssd_ctx* ctx, int rope_dim, float theta, int n_positions,
                              float* table_dev, void* s) {
    SSD_TRY(check_ctx(ctx));
    SSD_REQ(table_dev && rope_dim > 0 && rope_dim % 2 == 0 && n_positions > 0 && theta > 0.0f,
            SSD_ERR_ARG, "bad arguments");
    SSD_REQ(((uintptr_t)table_dev & 7u) == 0, SSD_ERR_ARG, "table not on an 8-byte boundary");
    k_paged_rope_table<<<n_positions, 128, 0, pick_stream(ctx, s)>>>((float2*)table_dev, rope_dim,
                                                                     theta);
    SSD_CK_LAUNCH();
    return SSD_OK;
}

extern "C" int ssd_paged_append(ssd_ctx* ctx, ssd_kv_cache* kv, const float* q, int64_t q_stride,
                                int n_head, const float* k, int64_t k_stride, const float* v,
                                int64_t v_stride, int n_rows, const float* q_norm,
                                const float* k_norm, float eps, const float* rope, int rope_dim,
                                int rope_positions, int rope_halves, const int32_t* pos,
                                const int32_t* seq, const int32_t* table, int n_seq,
                                int pages_per_seq, float* q_out, int64_t q_out_stride, void* s) {
    SSD_TRY(check_ctx(ctx));
    PagedAppendArgs a = {};
    SSD_TRY(paged_view(kv, table, n_seq, pages_per_seq, &a.v));
    SSD_REQ(n_rows >= 0 && n_head >= 0, SSD_ERR_ARG, "bad arguments");
    if (n_rows == 0) return SSD_OK;
    SSD_REQ(k && v && pos && (n_head == 0 || (q && q_out)), SSD_ERR_ARG, "null pointer");
    SSD_REQ(seq || n_rows <= n_seq, SSD_ERR_SHAPE, "%d rows without seq but %d sequences", n_rows,
            n_seq);
    const int64_t kvd = kv->kv_dim, qd = (int64_t)n_head * kv->head_dim;
    SSD_REQ(n_head % kv->n_head_kv == 0, SSD_ERR_SHAPE, "n_head %d not a multiple of n_head_kv %d",
            n_head, kv->n_head_kv);
    SSD_REQ(k_stride >= kvd && v_stride >= kvd && (n_head == 0 || (q_stride >= qd && q_out_stride >= qd)),
            SSD_ERR_SHAPE, "row strides shorter than the rows");
    if (rope) {
        SSD_REQ(rope_dim > 0 && rope_dim % 8 == 0 && rope_dim <= kv->head_dim, SSD_ERR_SHAPE,
                "rope_dim %d must be a multiple of 8 up to head_dim %d", rope_dim, kv->head_dim);
        SSD_REQ(rope_positions > 0, SSD_ERR_ARG, "empty rotation table");
        SSD_REQ(((uintptr_t)rope & 7u) == 0, SSD_ERR_ARG, "rotation table not on an 8-byte boundary");
    }
    a.q = q;
    a.k = k;
    a.x = v;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.x_stride = v_stride;
    a.n_head = n_head;
    a.n_rows = n_rows;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.rope = (const float2*)rope;
    a.rope_dim = rope_dim;
    a.rope_positions = rope_positions;
    a.rope_halves = rope_halves;
    a.pos = pos;
    a.seq = seq;
    a.q_out = q_out;
    a.q_out_stride = q_out_stride;
    a.status = ctx->dev_status;
    a.vec = aligned(q, q_stride, 4, 16) && aligned(k, k_stride, 4, 16) &&
            aligned(v, v_stride, 4, 16) && aligned(q_out, q_out_stride, 4, 16) &&
            aligned(q_norm, 0, 4, 16) && aligned(k_norm, 0, 4, 16) &&
            aligned(rope, 0, 4, 16);  // a position's row of the table is a multiple of 32 bytes
    return paged_dispatch(kv->paged_type, kv->head_dim,
                          AppendLaunch{a, pick_stream(ctx, s), ctx->pdl});
}

extern "C" int ssd_paged_read(ssd_ctx* ctx, const ssd_kv_cache* kv, int n_rows, const int32_t* pos,
                              const int32_t* seq, const int32_t* table, int n_seq,
                              int pages_per_seq, int out_type, void* k_out, int64_t k_stride,
                              void* v_out, int64_t v_stride, void* s) {
    SSD_TRY(check_ctx(ctx));
    PagedReadArgs a = {};
    SSD_TRY(paged_view(kv, table, n_seq, pages_per_seq, &a.v));
    SSD_REQ(out_type == SSD_TYPE_F32 || out_type == SSD_TYPE_F16 || out_type == SSD_TYPE_BF16,
            SSD_ERR_TYPE, "read-back type %d not supported (F32, F16, BF16)", out_type);
    SSD_REQ(n_rows >= 0, SSD_ERR_ARG, "bad arguments");
    if (n_rows == 0) return SSD_OK;
    SSD_REQ(pos && k_out && v_out, SSD_ERR_ARG, "null pointer");
    SSD_REQ(seq || n_rows <= n_seq, SSD_ERR_SHAPE, "%d rows without seq but %d sequences", n_rows,
            n_seq);
    SSD_REQ(k_stride >= kv->kv_dim && v_stride >= kv->kv_dim, SSD_ERR_SHAPE,
            "row strides shorter than the rows");
    const int e = out_type == SSD_TYPE_F32 ? 4 : 2;
    SSD_REQ((uintptr_t)k_out % e == 0 && (uintptr_t)v_out % e == 0, SSD_ERR_ARG,
            "output not aligned to its type");
    a.n_rows = n_rows;
    a.out_type = out_type;
    a.pos = pos;
    a.seq = seq;
    a.k = (uint8_t*)k_out;
    a.x = (uint8_t*)v_out;
    a.k_stride = k_stride;
    a.x_stride = v_stride;
    a.vec = aligned(k_out, k_stride, e, 4 * e) && aligned(v_out, v_stride, e, 4 * e);
    return paged_dispatch(kv->paged_type, kv->head_dim,
                          ReadLaunch{a, pick_stream(ctx, s), ctx->pdl});
}

extern "C" int ssd_paged_attention_workspace(ssd_ctx* ctx, const ssd_kv_cache* kv, size_t* bytes) {
    SSD_REQ(ctx && kv && bytes, SSD_ERR_ARG, "null pointer");
    SSD_REQ(kv->page_size > 0, SSD_ERR_STATE, "not a paged cache (ssd_kv_create_paged makes one)");
    *bytes = paged_attn_workspace(ctx, kv->head_dim);
    return SSD_OK;
}

extern "C" int ssd_paged_attention(ssd_ctx* ctx, const ssd_kv_cache* kv, const float* q,
                                   int64_t q_stride, int n_head, int n_rows, const int32_t* len,
                                   const int32_t* seq, const int32_t* table, int n_seq,
                                   int pages_per_seq, float scale, int window, float* out,
                                   int64_t out_stride, void* workspace, size_t workspace_bytes,
                                   void* s) {
    SSD_TRY(check_ctx(ctx));
    PagedAttnArgs a = {};
    SSD_TRY(paged_view(kv, table, n_seq, pages_per_seq, &a.v));
    SSD_REQ(n_rows >= 0 && window >= 0, SSD_ERR_ARG, "bad arguments");
    SSD_REQ(n_head > 0 && n_head % kv->n_head_kv == 0, SSD_ERR_SHAPE,
            "n_head %d not a multiple of n_head_kv %d", n_head, kv->n_head_kv);
    SSD_REQ(scale == scale && scale >= 0.0f, SSD_ERR_ARG, "scale must not be negative or NaN");
    if (n_rows == 0) return SSD_OK;
    SSD_REQ(q && len && out && workspace, SSD_ERR_ARG, "null pointer");
    SSD_REQ(((uintptr_t)workspace & 15u) == 0, SSD_ERR_ARG, "workspace not on a 16-byte boundary");
    const size_t need = paged_attn_workspace(ctx, kv->head_dim);
    SSD_REQ(workspace_bytes >= need, SSD_ERR_SHAPE, "workspace of %zu bytes, %zu needed",
            workspace_bytes, need);
    SSD_REQ(seq || n_rows <= n_seq, SSD_ERR_SHAPE, "%d rows without seq but %d sequences", n_rows,
            n_seq);
    const int64_t qd = (int64_t)n_head * kv->head_dim;
    SSD_REQ(q_stride >= qd && out_stride >= qd, SSD_ERR_SHAPE, "row strides shorter than the rows");
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.len = len;
    a.seq = seq;
    a.n_rows = n_rows;
    a.n_head = n_head;
    a.group = n_head / kv->n_head_kv;
    a.subs = (a.group + 7) / 8;
    a.window = window;
    a.scale = scale > 0.0f ? scale : 1.0f / sqrtf((float)kv->head_dim);
    a.work = (uint8_t*)workspace;
    a.status = ctx->dev_status;
    a.q_vec = aligned(q, q_stride, 4, 16);
    a.out_vec = aligned(out, out_stride, 4, 16);
    return launch_paged_attention(ctx, kv->paged_type, kv->head_dim, a, pick_stream(ctx, s),
                                  ctx->pdl);
}
