// Decode attention over 8-bit key/value pages (format: cache_8bit.cuh): segments of one token,
//   out = softmax(scale * q K^T) V,  K = 2^ek k8,  V = 2^ev v8,  keys lo .. pos (lo = pos - window + 1 with a window)
//
// All of it is memory traffic - each byte of a key or value is used for a handful of query heads - so the keys and values
// go straight from memory into the registers in which mma.sync wants them, in 16-byte pieces, and nothing is exchanged
// between the warps of a CTA until a piece of work ends.  A warp takes 64 keys (four blocks of 16) at a time:
//   S^T = K Q^T      m16n8k16, 16 keys x 8 query heads; the codes become half precision exactly (two instructions for four
//                    e4m3, five for int8), queries are scaled to [1, 2) per head so that half precision holds them
//   softmax          in 32 bits; a value block's scale joins the exponent: w = 2^(s + ev - m'), m' the running maximum of
//                    s + ev, so the weights of the second product are at most 1 whatever the scales are (half precision
//                    rounds them by 2^-12), and the sum of 2^(s - m') is kept beside it
//   O^T += V^T w^T   m16n8k16, 16 elements of the head x 8 query heads; movmatrix turns the weights, and V^T is what the
//                    pages hold
// The contractions do not care in which order keys or elements come, so the order is the one in which a lane's pieces lie:
//   keys     tile of 16 rows j = 0..3: row r holds token 4 j + (r & 1) + 2 (r >> 3) of block (r & 7) >> 1
//   elements lane t of a quad holds elements 64 c + 16 t .. + 15 of its rows, four of them per k step
//   tokens   lane t of a quad holds block t of each line of V^T, four tokens per k step j: those of the keys' tile j
//
// Work split: as in the tcgen05 decode kernel.  The 64-key tiles of all (request, kv head, eight query heads) triples form
// one sequence, `pair_cost` units before each, and every CTA (one per SM) takes an equal span of it.  A triple inside one
// span is finished by its CTA; a cut one leaves (maximum, sum, accumulator) per piece in the workspace, and the CTA that
// delivers its last missing piece adds the pieces up in the order of the keys.  Nothing waits for another CTA.  Within a
// piece the eight warps take tiles in turn and are added up in warp order through shared memory.
// A group of more than eight query heads is cut in pieces of eight, and its keys are read once for each (from L2 mostly).
#include <math.h>

#include "cache_8bit.cuh"

#define A8_WARPS 8
#define A8_THREADS (A8_WARPS * 32)
#define A8_TILE 64
#define A8_HEADS 8
#define A8_MAX_SEGS 1024
#define A8_SLOT_HEADS 16       // heads per slot of the workspace

struct A8Params {
    const bf16* q; int q_stride;
    const unsigned char* kcache; const unsigned char* vcache; const float* kscale; const float* vscale;
    const int* block_table; int bt_rows, bt_stride;
    const int* seg_off; const int* seg_slot; const int* seg_start; const int* seg_len;
    bf16* out;
    float* ws_acc; float* ws_ml; unsigned* ws_count;
    int num_pages, num_tokens, num_segments;
    int nq, nkv, group, head_tiles;      // head_tiles: eights of query heads per kv head
    int page_shift, window;
    int span_min, pair_cost;
    float scale_log2;
};

struct A8Piece {
    int seg, kvh, h0, heads, pos, lo, tile, ntiles;   // tile: first 64-key tile of the piece (absolute)
    int whole, slot, cta_first, pieces;
};

struct A8Cursor { int f, end, seg, span; };

__device__ __forceinline__ float a8_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void a8_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ unsigned a8_turn(unsigned x) {
    unsigned y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint4 a8_load(const unsigned char* p) {
    uint4 v;
    // not the read-only path: the pages were written by the kernel before this one, which may still have been running when
    // this kernel began
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ unsigned a8_word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// the newest position of a segment, kept within the block table
__device__ __forceinline__ int a8_pos(const A8Params& p, int seg) {
    const long long most = ((long long)p.bt_stride << p.page_shift) - 1;
    return (int)min((long long)p.seg_start[seg], most);
}
__device__ __forceinline__ int a8_lo(const A8Params& p, int pos) { return p.window > 0 ? max(0, pos - p.window + 1) : 0; }
__device__ __forceinline__ int a8_seg_tiles(const A8Params& p, int seg) {
    if (p.seg_len[seg] != 1) return 0;
    const int pos = a8_pos(p, seg);
    return pos < 0 ? 0 : pos / A8_TILE - a8_lo(p, pos) / A8_TILE + 1;
}
// pre[s]: tiles per triple of the segments before s, pre[A8_MAX_SEGS + 1 + s]: decoding segments before s
__device__ __forceinline__ int a8_seg_unit(const A8Params& p, const int* pre, int s) {
    return p.nkv * p.head_tiles * (pre[s] + p.pair_cost * pre[A8_MAX_SEGS + 1 + s]);
}

__device__ __forceinline__ void a8_begin(const A8Params& p, const int* pre, A8Cursor& c) {
    const int total = a8_seg_unit(p, pre, p.num_segments);
    c.span = max((total + (int)gridDim.x - 1) / (int)gridDim.x, p.span_min);
    const long long b = (long long)blockIdx.x * c.span;
    c.f = (int)(b < total ? b : total);
    c.end = (int)min((long long)c.f + c.span, (long long)total);
    int lo = 0, hi = p.num_segments;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a8_seg_unit(p, pre, mid) <= c.f) lo = mid; else hi = mid;
    }
    c.seg = lo;
}

__device__ __forceinline__ bool a8_next(const A8Params& p, const int* pre, A8Cursor& c, A8Piece& w) {
    while (c.f < c.end) {
        while (a8_seg_unit(p, pre, c.seg + 1) <= c.f) ++c.seg;       // ends: f lies before the end of the sequence
        const int n = pre[c.seg + 1] - pre[c.seg];
        const int per = n + p.pair_cost;
        const int rel = c.f - a8_seg_unit(p, pre, c.seg);
        const int tile0 = c.f - rel % per + p.pair_cost;              // unit of the triple's first tile
        const int lo_u = max(c.f, tile0), hi_u = min(c.end, tile0 + n);
        if (hi_u <= lo_u) { c.f = c.end; break; }                     // the span ends among the cost units
        const int triple = rel / per, ht = triple % p.head_tiles;
        w.seg = c.seg;
        w.kvh = triple / p.head_tiles;
        w.h0 = w.kvh * p.group + ht * A8_HEADS;
        w.heads = min(A8_HEADS, p.group - ht * A8_HEADS);
        w.pos = a8_pos(p, w.seg);
        w.lo = a8_lo(p, w.pos);
        w.tile = w.lo / A8_TILE + (lo_u - tile0);
        w.ntiles = hi_u - lo_u;
        w.whole = (lo_u == tile0 && hi_u == tile0 + n) ? 1 : 0;
        w.slot = lo_u == tile0 ? 1 : 0;
        w.cta_first = tile0 / c.span;
        w.pieces = (tile0 + n - 1) / c.span - w.cta_first + 1;
        c.f = hi_u;
        return true;
    }
    return false;
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(A8_THREADS, 1) attn_decode_8bit_kernel(const A8Params p) {
    constexpr int KC = D / 64;             // 16-byte pieces of a key row per lane
    constexpr int KS = D / 16;             // k steps of the first product, and 16-row tiles of V^T
    constexpr int LINE = D + 4;            // floats of a head's line in shared memory: no bank conflicts
    __shared__ int pre[2 * (A8_MAX_SEGS + 1)];
    __shared__ float part_o[A8_WARPS][A8_HEADS][LINE];
    __shared__ float part_m[A8_WARPS][A8_HEADS], part_l[A8_WARPS][A8_HEADS];
    __shared__ int last_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_trigger(PDL_ATTENTION);
    if (warp == 0) {
        int run = 0, run_d = 0;
        for (int s0 = 0; s0 < p.num_segments; s0 += 32) {
            const int s = s0 + lane;
            const int n = s < p.num_segments ? a8_seg_tiles(p, s) : 0, dflag = n > 0 ? 1 : 0;
            int inc = n, inc_d = dflag;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, inc, o), b = __shfl_up_sync(0xffffffffu, inc_d, o);
                if (lane >= o) { inc += a; inc_d += b; }
            }
            if (s < p.num_segments) { pre[s] = run + inc - n; pre[A8_MAX_SEGS + 1 + s] = run_d + inc_d - dflag; }
            run += __shfl_sync(0xffffffffu, inc, 31);
            run_d += __shfl_sync(0xffffffffu, inc_d, 31);
        }
        if (lane == 0) { pre[p.num_segments] = run; pre[A8_MAX_SEGS + 1 + p.num_segments] = run_d; }
    }
    __syncthreads();
    A8Cursor cur;
    a8_begin(p, pre, cur);
    A8Piece w, cut[2];
    int num_cut = 0;
    const int page_blocks = 1 << (p.page_shift - 4);
    while (a8_next(p, pre, cur, w)) {
        const int slot = p.seg_slot[w.seg];
        const bool has_row = slot >= 0 && slot < p.bt_rows;
        const int* table = p.block_table + (size_t)(has_row ? slot : 0) * p.bt_stride;
        // block (lane >> 3) of a tile: its number in the pool, -1 if it holds no visible key or has no page
        auto lookup = [&](int tile) -> int {
            const int key = tile * A8_TILE + (lane >> 3) * C8_BLOCK;
            if (!has_row || tile >= w.tile + w.ntiles || key > w.pos || key + C8_BLOCK <= w.lo) return -1;
            const int page = table[key >> p.page_shift];
            if (page < 0 || page >= p.num_pages) return -1;
            return (page * p.nkv + w.kvh) * page_blocks + ((key & ((1 << p.page_shift) - 1)) >> 4);
        };
        uint4 kr[4][2][KC], vr[KS][2];
        float ks = 0.0f, vs = 0.0f, ks_next, vs_next;
        auto load_k = [&](int id) {       // a block that is not there: block 0 is loaded and masked
            const unsigned char* base = p.kcache + (size_t)max(id, 0) * (C8_BLOCK * D) + (g & 1) * D + 16 * t;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < KC; ++c) kr[j][h][c] = a8_load(base + (4 * j + 2 * h) * D + 64 * c);
        };
        auto load_v = [&](int id) {       // id: of block t
            const unsigned char* base = p.vcache + (size_t)max(id, 0) * (C8_BLOCK * D) + g * C8_BLOCK;
#pragma unroll
            for (int m = 0; m < KS; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) vr[m][h] = a8_load(base + (16 * m + 8 * h) * C8_BLOCK);
        };
        const int first = w.tile + warp, stop = w.tile + w.ntiles;
        int id = lookup(first), id_next = lookup(first + A8_WARPS);
        if (first < stop) {
            load_k(id);
            load_v(__shfl_sync(0xffffffffu, id, 8 * t));
            ks = p.kscale[max(id, 0)]; vs = p.vscale[max(id, 0)];
        }
        // queries of head g as the second operand, scaled by a power of two into [1, 2); lanes of heads that are not: zeros
        unsigned qb[KS][2];
        float f0, f1;
        {
            const int row = p.seg_off[w.seg];
            const bool live = g < w.heads && row >= 0 && row < p.num_tokens;
            const bf16* src = p.q + (size_t)(live ? row : 0) * p.q_stride + (size_t)(w.h0 + (live ? g : 0)) * D + 16 * t;
            uint4 raw[KC][2];
            float amax = 0.0f;
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    raw[c][h] = live ? *reinterpret_cast<const uint4*>(src + 64 * c + 8 * h) : make_uint4(0u, 0u, 0u, 0u);
                    const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&raw[c][h]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(fabsf(__low2float(x[i])), fabsf(__high2float(x[i]))));
                }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int e = max(-120, min(120, (int)(__float_as_uint(amax) >> 23) - 127));
            const float down = c8_pow2(-e);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                // k step: elements 64 c + 16 t + 4 i .. + 3 with c = k / 4, i = k % 4
                const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&raw[k / 4][(k % 4) / 2]) + 2 * (k % 2);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const __half2 v = __floats2half2_rn(__low2float(x[h]) * down, __high2float(x[h]) * down);
                    qb[k][h] = *reinterpret_cast<const unsigned*>(&v);
                }
            }
            const float up = p.scale_log2 * c8_pow2(e);
            f0 = __shfl_sync(0xffffffffu, up, 8 * t);          // heads 2t and 2t + 1
            f1 = __shfl_sync(0xffffffffu, up, 8 * t + 4);
        }
        float o[KS][4];
#pragma unroll
        for (int m = 0; m < KS; ++m) { o[m][0] = 0.0f; o[m][1] = 0.0f; o[m][2] = 0.0f; o[m][3] = 0.0f; }
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

#pragma unroll 1
        for (int tile = first; tile < stop; tile += A8_WARPS) {
            const int id_after = lookup(tile + 2 * A8_WARPS);
            const bool more = tile + A8_WARPS < stop;
            ks_next = 0.0f; vs_next = 0.0f;
            float s[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[j][0] = 0.0f; s[j][1] = 0.0f; s[j][2] = 0.0f; s[j][3] = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    unsigned a0, a1, a2, a3;
                    c8_decode4<E4M3>(a8_word(kr[j][0][k / 4], k % 4), a0, a2);
                    c8_decode4<E4M3>(a8_word(kr[j][1][k / 4], k % 4), a1, a3);
                    a8_mma(s[j], a0, a1, a2, a3, qb[k][0], qb[k][1]);
                }
            }
            if (more) {
                load_k(id_next);
                ks_next = p.kscale[max(id_next, 0)]; vs_next = p.vscale[max(id_next, 0)];
            }
            // ---- softmax: all rows of a lane lie in block g >> 1 -------------------------------------------------
            const int base = tile * A8_TILE;
            const bool full = base >= w.lo && base + A8_TILE - 1 <= w.pos && __all_sync(0xffffffffu, id >= 0);
            vs = fmaxf(vs, 8.673617379884035e-19f);      // 2^-60: a scale of zero still counts in the sum
            const float lv = log2f(vs), c0 = f0 * ks, c1 = f1 * ks;
            float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float a = s[j][2 * h] * c0, b = s[j][2 * h + 1] * c1;
                    if (!full) {
                        const int key = base + (g >> 1) * C8_BLOCK + 4 * j + 2 * h + (g & 1);
                        if (id < 0 || key < w.lo || key > w.pos) { a = -INFINITY; b = -INFINITY; }
                    }
                    s[j][2 * h] = a; s[j][2 * h + 1] = b;
                    x0 = fmaxf(x0, a); x1 = fmaxf(x1, b);
                }
            }
            // a block that is not there has no scale: its lanes' maxima are already -inf
            if (id >= 0) { x0 += lv; x1 += lv; }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
            }
            const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
            if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
                const float r0 = m0 == -INFINITY ? 0.0f : a8_ex2(m0 - n0), r1 = m1 == -INFINITY ? 0.0f : a8_ex2(m1 - n1);
                l0 *= r0; l1 *= r1;
#pragma unroll
                for (int m = 0; m < KS; ++m) { o[m][0] *= r0; o[m][1] *= r1; o[m][2] *= r0; o[m][3] *= r1; }
                m0 = n0; m1 = n1;
            }
            const float e0 = id >= 0 ? (m0 == -INFINITY ? 0.0f : m0) - lv : 0.0f, e1 = id >= 0 ? (m1 == -INFINITY ? 0.0f : m1) - lv : 0.0f;
            const float back = id >= 0 ? 1.0f / vs : 0.0f;
            unsigned pb[4][2];
            float t0 = 0.0f, t1 = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float a = a8_ex2(s[j][2 * h] - e0), b = a8_ex2(s[j][2 * h + 1] - e1);
                    t0 += a; t1 += b;
                    const __half2 v = __floats2half2_rn(a, b);
                    pb[j][h] = a8_turn(*reinterpret_cast<const unsigned*>(&v));
                }
            l0 = fmaf(t0, back, l0); l1 = fmaf(t1, back, l1);
            if (!full) {                   // whatever lies in the value bytes of hidden keys must not meet a weight of zero
                const int begin = base + t * C8_BLOCK;
                const bool there = __shfl_sync(0xffffffffu, id, 8 * t) >= 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    unsigned mask = 0u;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int key = begin + 4 * j + b;
                        mask |= (there && key >= w.lo && key <= w.pos) ? 0xffu << (8 * b) : 0u;
                    }
#pragma unroll
                    for (int m = 0; m < KS; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (j == 0) vr[m][h].x &= mask; else if (j == 1) vr[m][h].y &= mask;
                            else if (j == 2) vr[m][h].z &= mask; else vr[m][h].w &= mask;
                        }
                }
            }
#pragma unroll
            for (int m = 0; m < KS; ++m) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    unsigned a0, a1, a2, a3;
                    c8_decode4<E4M3>(a8_word(vr[m][0], j), a0, a2);
                    c8_decode4<E4M3>(a8_word(vr[m][1], j), a1, a3);
                    a8_mma(o[m], a0, a1, a2, a3, pb[j][0], pb[j][1]);
                }
            }
            if (more) load_v(__shfl_sync(0xffffffffu, id_next, 8 * t));
            id = id_next; id_next = id_after; ks = ks_next; vs = vs_next;
        }
        // ---- the warps' shares of the piece, added up in warp order ---------------------------------------------------
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) { l0 += __shfl_xor_sync(0xffffffffu, l0, d); l1 += __shfl_xor_sync(0xffffffffu, l1, d); }
        if (g == 0) {
            part_m[warp][2 * t] = m0; part_m[warp][2 * t + 1] = m1;
            part_l[warp][2 * t] = l0; part_l[warp][2 * t + 1] = l1;
        }
#pragma unroll
        for (int m = 0; m < KS; ++m) {
            part_o[warp][2 * t][16 * m + g] = o[m][0]; part_o[warp][2 * t + 1][16 * m + g] = o[m][1];
            part_o[warp][2 * t][16 * m + 8 + g] = o[m][2]; part_o[warp][2 * t + 1][16 * m + 8 + g] = o[m][3];
        }
        __syncthreads();
        const int row = p.seg_off[w.seg];
        for (int i = threadIdx.x; i < w.heads * D; i += A8_THREADS) {
            const int h = i / D, e = i % D;
            float top = -INFINITY, sum = 0.0f, den = 0.0f;
#pragma unroll
            for (int x = 0; x < A8_WARPS; ++x) top = fmaxf(top, part_m[x][h]);
            const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int x = 0; x < A8_WARPS; ++x) {
                const float f = a8_ex2(part_m[x][h] - ref);
                sum = fmaf(f, part_o[x][h][e], sum);
                den = fmaf(f, part_l[x][h], den);
            }
            if (w.whole) {
                if (row >= 0 && row < p.num_tokens)
                    p.out[((size_t)row * p.nq + w.h0 + h) * D + e] = __float2bfloat16_rn(den == 0.0f ? 0.0f : sum / den);
            } else {
                const size_t at = ((size_t)blockIdx.x * 2 + w.slot) * A8_SLOT_HEADS + h;
                p.ws_acc[at * D + e] = sum;
                if (e == 0) { p.ws_ml[at * 2] = top; p.ws_ml[at * 2 + 1] = den; }
            }
        }
        if (!w.whole) cut[num_cut++] = w;
        __syncthreads();
    }
    // ---- pieces of cut triples: reported when the span is done ---------------------------------------------------------
    for (int c = 0; c < num_cut; ++c) {
        const A8Piece& z = cut[c];
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            const unsigned before = atomicAdd(&p.ws_count[z.cta_first], 1u);
            last_flag = before + 1 == (unsigned)z.pieces;
            if (last_flag) p.ws_count[z.cta_first] = 0u;          // zero for the next launch
            __threadfence();
        }
        __syncthreads();
        if (!last_flag) continue;
        const int row = p.seg_off[z.seg];
        for (int i = threadIdx.x; i < z.heads * D; i += A8_THREADS) {
            const int h = i / D, e = i % D;
            float top = -INFINITY, sum = 0.0f, den = 0.0f;
            for (int x = 0; x < z.pieces; ++x) {                  // the first piece lies in slot 1 of its CTA, the others in slot 0
                const size_t at = ((size_t)(z.cta_first + x) * 2 + (x == 0 ? 1 : 0)) * A8_SLOT_HEADS + h;
                const float m = __ldcg(&p.ws_ml[at * 2]), l = __ldcg(&p.ws_ml[at * 2 + 1]), a = __ldcg(&p.ws_acc[at * D + e]);
                const float n = fmaxf(top, m), ref = n == -INFINITY ? 0.0f : n;
                const float old = a8_ex2(top - ref), now = a8_ex2(m - ref);
                sum = sum * old + a * now;
                den = den * old + l * now;
                top = n;
            }
            if (row >= 0 && row < p.num_tokens)
                p.out[((size_t)row * p.nq + z.h0 + h) * D + e] = __float2bfloat16_rn(den == 0.0f ? 0.0f : sum / den);
        }
        __syncthreads();
    }
}

PI_EXPORT int pi_attention_decode_8bit(const void* q, int q_stride, const void* kcache, const void* vcache, const float* kscale,
                                       const float* vscale, int cache_dtype, long long num_pages, const int* block_table, int bt_rows,
                                       int bt_stride, const int* seg_off, const int* seg_slot, const int* seg_start,
                                       const int* seg_len, void* out, float* ws_acc, float* ws_ml, void* ws_count, int ws_ctas,
                                       int span_min, int pair_cost, int num_tokens, int num_segments, int nq, int nkv, int head_dim,
                                       int page_size, int window, float scale, cudaStream_t stream) {
    if (num_segments <= 0 || num_tokens <= 0) return 0;
    if (head_dim != 64 && head_dim != 128) return pi_refuse("pi_attention_decode_8bit: head size %d is not 64 or 128", head_dim);
    if (!(scale > 0.0f)) return pi_refuse("pi_attention_decode_8bit: the score scale must be positive");
    if (nq <= 0 || nkv <= 0 || nq % nkv != 0) return pi_refuse("pi_attention_decode_8bit: nq=%d must be a positive multiple of nkv=%d", nq, nkv);
    if (num_segments > A8_MAX_SEGS) return pi_refuse("pi_attention_decode_8bit: %d segments; this kernel takes at most %d", num_segments, A8_MAX_SEGS);
    if (page_size < C8_BLOCK || (page_size & (page_size - 1))) return pi_refuse("pi_attention_decode_8bit: page size %d must be a power of two of at least 16", page_size);
    if (cache_dtype != PI_E4M3 && cache_dtype != PI_INT8) return pi_refuse("pi_attention_decode_8bit: unknown dtype code %d of the pages", cache_dtype);
    if (window < 0 || bt_rows <= 0 || bt_stride <= 0) return pi_refuse("pi_attention_decode_8bit: window=%d, block table [%d, %d]", window, bt_rows, bt_stride);
    if (ws_ctas <= 0 || ws_acc == nullptr || ws_ml == nullptr || ws_count == nullptr) return pi_refuse("pi_attention_decode_8bit: the workspace is missing");
    if (span_min < 1 || pair_cost < 0 || pair_cost > 64) return pi_refuse("pi_attention_decode_8bit: span_min=%d must be at least 1 and pair_cost=%d between 0 and 64", span_min, pair_cost);
    if (q_stride % 8 != 0 || (((uintptr_t)q | (uintptr_t)kcache | (uintptr_t)vcache) & 15))
        return pi_refuse("pi_attention_decode_8bit: q and the pages must start on 16-byte boundaries, q with a stride that is a multiple of 8");
    const long long blocks = num_pages * nkv * (page_size / C8_BLOCK);
    if (num_pages <= 0 || blocks > 2147483647LL) return pi_refuse("pi_attention_decode_8bit: %lld pages are %lld blocks: beyond the limit", num_pages, blocks);
    if ((long long)bt_stride * page_size > 2147483647LL - 2 * A8_TILE * A8_WARPS * 4)
        return pi_refuse("pi_attention_decode_8bit: block tables of %d pages are beyond the limit", bt_stride);
    A8Params p;
    p.q = (const bf16*)q; p.q_stride = q_stride;
    p.kcache = (const unsigned char*)kcache; p.vcache = (const unsigned char*)vcache; p.kscale = kscale; p.vscale = vscale;
    p.block_table = block_table; p.bt_rows = bt_rows; p.bt_stride = bt_stride;
    p.seg_off = seg_off; p.seg_slot = seg_slot; p.seg_start = seg_start; p.seg_len = seg_len;
    p.out = (bf16*)out; p.ws_acc = ws_acc; p.ws_ml = ws_ml; p.ws_count = (unsigned*)ws_count;
    p.num_pages = (int)num_pages; p.num_tokens = num_tokens; p.num_segments = num_segments;
    p.nq = nq; p.nkv = nkv; p.group = nq / nkv; p.head_tiles = (p.group + A8_HEADS - 1) / A8_HEADS;
    p.window = window; p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.span_min = span_min; p.pair_cost = pair_cost;
    p.scale_log2 = scale * 1.4426950408889634f;
    long long seg_tiles = ((long long)bt_stride * page_size + A8_TILE - 1) / A8_TILE;
    if (window > 0 && seg_tiles > window / A8_TILE + 2) seg_tiles = window / A8_TILE + 2;
    const long long units = (long long)num_segments * nkv * p.head_tiles * (seg_tiles + pair_cost);
    if (units > 1000000000LL) return pi_refuse("pi_attention_decode_8bit: up to %lld tiles of keys are beyond the limit", units);
    const dim3 grid((unsigned)ws_ctas), threads(A8_THREADS);
    if (head_dim == 128) {
        if (cache_dtype == PI_E4M3) pi_launch(attn_decode_8bit_kernel<128, true>, grid, threads, 0, stream, p);
        else pi_launch(attn_decode_8bit_kernel<128, false>, grid, threads, 0, stream, p);
    } else {
        if (cache_dtype == PI_E4M3) pi_launch(attn_decode_8bit_kernel<64, true>, grid, threads, 0, stream, p);
        else pi_launch(attn_decode_8bit_kernel<64, false>, grid, threads, 0, stream, p);
    }
    return pi_check_launch("pi_attention_decode_8bit");
}
