// Writing and reading back the 8-bit key/value pages (format: cache_8bit.cuh).
#include "cache_8bit.cuh"

// ---------------------------------------------------------------------------------------------------
// Per-head RMSNorm + rotation of queries and keys, keys and values into their 8-bit pages.
// Input: qkv [T, row_stride] bf16 holding nq query heads, nkv key heads, nkv value heads of width D per token.
//   query head   q / sqrt(mean q^2 + eps) * qw, rotated, to q_out [T, nq * D] bf16
//   key head     the same with kw, rounded to bf16 (what a bf16 page would hold), then encoded
//   value head   encoded as it is
// slot_map[t] = pool slot (page * page_size + place in the page) of token t; a slot outside the pool is counted in
// *error_count, once per key and value head, and skipped.  Tokens that follow one another in slot order and share a block
// form a run; a run that starts at the block's first token begins the block anew (the rest of it becomes zeros), another
// one adds to it: the scale is kept or raised, and if it is raised the tokens that lie there are encoded again.  The runs
// of a call must lie in distinct blocks.
// Not-a-number keys and values are stored as zero and infinities as the largest number of the format, so a page never
// holds what would spread from a masked place (0 x NaN).
//
// A block of four warps takes one key or value head of a run: the scale needs the whole run, at most 16 rows of D elements.
// Lanes of D / 8 form a group that takes 16-byte pieces of one or two rows, so everything a run needs (rows, rotation, what lies
// in the block) is asked for at once: the kernel is a chain of two round trips, the slots and the rest.  (One warp for all 16
// rows went through the rotation tables of eight rows one after the other: 25 us where this form took 12, before keys kept their
// rounding errors; it takes 15.5 now.)  A block looks for the
// runs that begin among `window` tokens: 16 in a step of many tokens - one run, as a rule - and 1 in a decode step.  Query heads
// are plain streaming work; in a step of many tokens they are a kernel of their own, in a small one part of the same launch.
// Measured (B200, 32 + 8 + 8 heads of 128, pairs of neighbours): 19.4 (e4m3) to 20.6 us (int8) for 2,045 tokens, both kernels,
// 46 MB (2.2 TB/s: too few loads in flight per warp, as in the bf16 kernel, and the arithmetic of the keys); 3.1 us for 8
// decoding requests.  Pairs of halves: 23.8 to 24.4 and 4.0 us; a lane then holds eight cosines and sines for each of its rows, and
// 17 words of it are spilled from the 80 registers that six blocks per SM leave.
// ---------------------------------------------------------------------------------------------------
#define CW_WARPS 4
#define CW_Q_ROWS 4          // query rows in flight per lane group
#define CW_SMALL 128         // tokens up to which one launch does everything, a window of one token per block

struct CwParams {
    const bf16* qkv; int row_stride;
    const void* qw; const void* kw; int wide; float eps; int has_norm;      // wide: the weights are float
    const float* cos_t; const float* sin_t; int rot_pairs;
    unsigned char* kcache; unsigned char* vcache; float* kscale; float* vscale;
    const long long* slot_map; long long num_slots; int page_shift;
    bf16* q_out;
    int nq, nkv, num_tokens;
    int window;                       // tokens among which a block looks for the beginnings of runs: 1 or 16
    long long kv_units;               // blocks' worth of keys and values
    int q_shares;                     // warps' worth of a token's query heads
    int* error_count;
};

__device__ __forceinline__ void cw_unpack(const uint4& raw, float (&x)[8]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __low2float(h[i]); x[2 * i + 1] = __high2float(h[i]); }
}
__device__ __forceinline__ uint4 cw_pack(const float (&x)[8]) {
    uint4 raw;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    return raw;
}

// 8 norm weights from element 8 * sub on
__device__ __forceinline__ void cw_weights(const void* w, int wide, int sub, float (&v)[8]) {
    if (!wide) {
        cw_unpack(reinterpret_cast<const uint4*>(w)[sub], v);
    } else {
        const float4 a = reinterpret_cast<const float4*>(w)[2 * sub], b = reinterpret_cast<const float4*>(w)[2 * sub + 1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
}

// what the rotation of one row needs, for the 8 elements of a lane: asked for ahead of use
template <bool ADJ> struct CwTurn { float c[ADJ ? 4 : 8], s[ADJ ? 4 : 8]; };

template <int D, bool ADJ>
__device__ __forceinline__ void cw_turn_load(const CwParams& p, int t, int sub, CwTurn<ADJ>& r) {
    if (p.rot_pairs == 0) return;
    const size_t row = (size_t)t * p.rot_pairs;
    if constexpr (ADJ) {                                 // pairs (2i, 2i + 1); rot_pairs is a multiple of 4
        if (4 * sub < p.rot_pairs) {
            *reinterpret_cast<float4*>(r.c) = *reinterpret_cast<const float4*>(p.cos_t + row + 4 * sub);
            *reinterpret_cast<float4*>(r.s) = *reinterpret_cast<const float4*>(p.sin_t + row + 4 * sub);
        }
    } else {                                            // pairs (i, i + rot_pairs); rot_pairs is a multiple of 8
        const int shift = p.rot_pairs / 8;
        if (sub < 2 * shift) {
            const int at = 8 * (sub < shift ? sub : sub - shift);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                *reinterpret_cast<float4*>(r.c + 4 * q) = *reinterpret_cast<const float4*>(p.cos_t + row + at + 4 * q);
                *reinterpret_cast<float4*>(r.s + 4 * q) = *reinterpret_cast<const float4*>(p.sin_t + row + at + 4 * q);
            }
        }
    }
}

// norm and rotation of one row spread over D / 8 lanes; every lane of the warp calls it (x of rows that do not exist: zeros)
template <int D, bool ADJ>
__device__ __forceinline__ void cw_norm_rope(const CwParams& p, int sub, const float (&w)[8], const CwTurn<ADJ>& r, float (&x)[8]) {
    constexpr int LANES = D / 8;
    if (p.has_norm) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) ss += x[i] * x[i] + x[i + 1] * x[i + 1];
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = 1.0f / sqrtf(ss / (float)D + p.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[i];
    }
    if (p.rot_pairs == 0) return;
    if constexpr (ADJ) {
        if (4 * sub < p.rot_pairs) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const float r0 = x[2 * h] * r.c[h] - x[2 * h + 1] * r.s[h], r1 = x[2 * h] * r.s[h] + x[2 * h + 1] * r.c[h];
                x[2 * h] = r0; x[2 * h + 1] = r1;
            }
        }
    } else {
        const int shift = p.rot_pairs / 8;              // the partner's lane
        const bool first = sub < shift, second = !first && sub < 2 * shift;
        const int partner = first ? sub + shift : second ? sub - shift : sub;
        float other[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xffffffffu, x[i], partner, LANES);
        if (first || second) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = first ? x[i] * r.c[i] - other[i] * r.s[i] : other[i] * r.s[i] + x[i] * r.c[i];
        }
    }
}

// a c + b s of numbers that are sums a + al and b + bl, as such a sum: rounding errors of products and sum are kept
__device__ __forceinline__ float2 cw_dot2(float2 a, float c, float2 b, float s) {
    // (intrinsics: nothing is to be drawn together here)
    const float m = __fmul_rn(a.x, c), n = __fmul_rn(b.x, s), h = __fadd_rn(m, n), t = __fsub_rn(h, m);
    const float sum_err = __fadd_rn(__fsub_rn(m, __fsub_rn(h, t)), __fsub_rn(n, t));
    return make_float2(h, sum_err + (fmaf(a.x, c, -m) + fmaf(b.x, s, -n)) + fmaf(a.y, c, b.y * s));
}

// cw_norm_rope for a key row, to bf16.  A key is rounded to bf16 and then to its code, and one that lies close to the middle
// between two codes falls to the other one if the errors before reach across it.  So the roundings of the norm and the rotation
// are kept beside the value until its end: of 34 million keys none has another code than by the formula in 64 bits; with one
// rounding after the other 21 had (19 with 32-bit arithmetic in torch).  It costs 2.6 us of 20.6 for 2,045 tokens.
template <int D, bool ADJ>
__device__ __forceinline__ uint4 cw_key_row(const CwParams& p, int sub, const float (&w)[8], const CwTurn<ADJ>& r, const uint4& raw) {
    constexpr int LANES = D / 8;
    float x[8];
    cw_unpack(raw, x);
    float2 v[8];
    float inv = 1.0f, inv_err = 0.0f;
    if (p.has_norm) {
        float ss = 0.0f, ss_err = 0.0f;                      // the sum of squares and what its roundings left out
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float n = fmaf(x[k], x[k], ss);
            ss_err += fmaf(x[k], x[k], __fsub_rn(ss, n));
            ss = n;
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, ss, o), n = __fadd_rn(ss, other), t = __fsub_rn(n, ss);
            ss_err += __shfl_xor_sync(0xffffffffu, ss_err, o);
            ss_err += __fadd_rn(__fsub_rn(ss, __fsub_rn(n, t)), __fsub_rn(other, t));
            ss = n;
        }
        const float mean = ss * (1.0f / D), a = __fadd_rn(mean, p.eps), d = __fsub_rn(a, mean);
        const float a_err = __fadd_rn(__fsub_rn(mean, __fsub_rn(a, d)), __fsub_rn(p.eps, d)) + ss_err * (1.0f / D);
        inv = rsqrtf(a);
        const float t = __fmul_rn(a, inv);                   // a step of Newton's: inv (1 + (1 - (a + a_err) inv^2) / 2)
        inv_err = 0.5f * inv * (fmaf(-t, inv, 1.0f) - (fmaf(a, inv, -t) + a_err * inv) * inv);
        if (!(fabsf(inv_err) <= inv)) inv_err = 0.0f;        // a is infinite, zero or no number
#pragma unroll
        for (int i = 0; i < 8; ++i) { v[i].x = __fmul_rn(x[i], w[i]); v[i].y = fmaf(x[i], w[i], -v[i].x); }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = make_float2(x[i], 0.0f);
    }
    if (p.rot_pairs > 0) {
        if constexpr (ADJ) {
            if (4 * sub < p.rot_pairs) {
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const float2 u = cw_dot2(v[2 * h], r.c[h], v[2 * h + 1], -r.s[h]);
                    v[2 * h + 1] = cw_dot2(v[2 * h], r.s[h], v[2 * h + 1], r.c[h]);
                    v[2 * h] = u;
                }
            }
        } else {
            const int shift = p.rot_pairs / 8;
            const bool first = sub < shift, second = !first && sub < 2 * shift;
            const int partner = first ? sub + shift : second ? sub - shift : sub;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 other = make_float2(__shfl_sync(0xffffffffu, v[i].x, partner, LANES), __shfl_sync(0xffffffffu, v[i].y, partner, LANES));
                if (first || second) v[i] = cw_dot2(v[i], r.c[i], other, first ? -r.s[i] : r.s[i]);
            }
        }
    }
    uint4 out;
    unsigned* half = reinterpret_cast<unsigned*>(&out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float e[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float2 u = v[2 * i + k];
            const float m = __fmul_rn(u.x, inv);
            float err = fmaf(u.x, inv, -m) + fmaf(u.x, inv_err, u.y * inv);
            if (!(fabsf(err) <= fabsf(m))) err = 0.0f;       // of infinities
            e[k] = m + err;
        }
        const __nv_bfloat162 pair = __floats2bfloat162_rn(e[0], e[1]);
        half[i] = *reinterpret_cast<const unsigned*>(&pair);
    }
    return out;
}

// element i (0..7) of four registers of bf16 pairs
__device__ __forceinline__ float cw_element(const uint4& raw, int i) {
    const unsigned w = i < 2 ? raw.x : i < 4 ? raw.y : i < 6 ? raw.z : raw.w;
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
}

// query heads: a warp takes CW_Q_ROWS per lane group of one token, so that one piece of the rotation tables does for all
template <int D, bool ADJ>
__device__ __forceinline__ void cw_queries(const CwParams& p, unsigned unit) {
    constexpr int LANES = D / 8, GROUPS = 32 / LANES;
    const int lane = threadIdx.x & 31, sub = lane % LANES, grp = lane / LANES;
    const unsigned t = unit / (unsigned)p.q_shares;
    if (t >= (unsigned)p.num_tokens) return;
    const int head0 = (int)(unit - t * p.q_shares) * GROUPS * CW_Q_ROWS + grp;
    const bf16* src = p.qkv + (size_t)t * p.row_stride;
    bf16* dst = p.q_out + (size_t)t * p.nq * D;
    uint4 raw[CW_Q_ROWS];
#pragma unroll
    for (int j = 0; j < CW_Q_ROWS; ++j)
        raw[j] = head0 + j * GROUPS < p.nq ? reinterpret_cast<const uint4*>(src + (head0 + j * GROUPS) * D)[sub] : make_uint4(0u, 0u, 0u, 0u);
    float w[8];
    if (p.has_norm) cw_weights(p.qw, p.wide, sub, w);
    CwTurn<ADJ> turn;
    cw_turn_load<D, ADJ>(p, (int)t, sub, turn);
#pragma unroll
    for (int j = 0; j < CW_Q_ROWS; ++j) {
        float x[8];
        cw_unpack(raw[j], x);
        cw_norm_rope<D, ADJ>(p, sub, w, turn, x);
        if (head0 + j * GROUPS < p.nq) reinterpret_cast<uint4*>(dst + (head0 + j * GROUPS) * D)[sub] = cw_pack(x);
    }
}

template <int D>
struct CwShared {
    float amax[CW_WARPS];
    unsigned tile[D][5];          // a value block on its way to its transposed place: 16 bytes a line, padded
};

// the run of `count` tokens that begins with token t, in one block of one key or value head (which: key heads, then value
// heads); the whole thread block
template <int D, bool ADJ, bool E4M3>
__device__ __forceinline__ void cw_run(const CwParams& p, CwShared<D>& sh, int t, long long slot, int count, int which) {
    constexpr int LANES = D / 8, GROUPS = 32 / LANES, ROWS = C8_BLOCK / CW_WARPS / GROUPS;       // D 128: 2 rows a lane; 64: 1
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LANES, grp = lane / LANES;
    const bool is_v = which >= p.nkv;
    const int head = is_v ? which - p.nkv : which;
    const int off = (int)(slot & (C8_BLOCK - 1));
    const int page_blocks = 1 << (p.page_shift - 4);
    const long long page = slot >> p.page_shift;
    const long long block = (page * p.nkv + head) * page_blocks + (((int)slot & ((1 << p.page_shift) - 1)) >> 4);
    unsigned char* data = (is_v ? p.vcache : p.kcache) + (size_t)block * C8_BLOCK * D;
    float* scale = (is_v ? p.vscale : p.kscale) + block;
    const int row0 = (warp * GROUPS + grp) * ROWS;                                      // the lane's rows of the block

    // everything that is read, at once
    const bf16* src = p.qkv + (size_t)t * p.row_stride + (size_t)(p.nq + which) * D;
    uint4 row[ROWS];
    CwTurn<ADJ> turn[ROWS];
    uint2 old_k[ROWS];
    uint4 old_v = make_uint4(0u, 0u, 0u, 0u);
    const float old_scale = off > 0 ? *scale : 0.0f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int i = row0 + r - off;                                                   // token t + i
        const bool fresh = i >= 0 && i < count;
        row[r] = fresh ? reinterpret_cast<const uint4*>(src + (size_t)i * p.row_stride)[sub] : make_uint4(0u, 0u, 0u, 0u);
        old_k[r] = make_uint2(0u, 0u);
        if (!is_v) {
            cw_turn_load<D, ADJ>(p, t + max(0, min(i, count - 1)), sub, turn[r]);
            if (!fresh && off > 0) old_k[r] = reinterpret_cast<const uint2*>(data + (row0 + r) * D)[sub];
        }
    }
    if (is_v && off > 0 && threadIdx.x < D) old_v = reinterpret_cast<const uint4*>(data)[threadIdx.x];
    if (!is_v) {
        float w[8];
        if (p.has_norm) cw_weights(p.kw, p.wide, sub, w);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int i = row0 + r - off;
            const uint4 key = cw_key_row<D, ADJ>(p, sub, w, turn[r], row[r]);
            if (i >= 0 && i < count) row[r] = key;
        }
    }
    float amax = 0.0f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(cw_element(row[r], i)));     // fmaxf passes over NaN
    }
    amax = warp_max(amax);
    if (lane == 0) sh.amax[warp] = amax;
    __syncthreads();                                      // (also: every thread has read the old scale)
#pragma unroll
    for (int x = 0; x < CW_WARPS; ++x) amax = fmaxf(amax, sh.amax[x]);
    int e = c8_exponent<E4M3>(amax), e_old = e;
    if (off > 0) { e_old = c8_scale_exponent(old_scale); e = max(e, e_old); }
    const bool again = off > 0 && e != e_old;             // what lies in the block is encoded again
    const float inv = c8_pow2(-e), shrink = c8_pow2(e_old - e);
    if (threadIdx.x == 0 && (off == 0 || again)) *scale = c8_pow2(e);
    auto coded = [&](float a, float b) -> unsigned {
        a = a == a ? a * inv : 0.0f;
        b = b == b ? b * inv : 0.0f;
        return c8_encode2<E4M3>(a, b);
    };
    auto shrunk = [&](unsigned codes) -> unsigned {       // four old codes at the new scale
        const float2 a = __half22float2(c8_decode2<E4M3>(codes & 0xffffu)), b = __half22float2(c8_decode2<E4M3>(codes >> 16));
        return c8_encode2<E4M3>(a.x * shrink, a.y * shrink) | (c8_encode2<E4M3>(b.x * shrink, b.y * shrink) << 16);
    };
    uint2 code[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        code[r].x = coded(cw_element(row[r], 0), cw_element(row[r], 1)) | (coded(cw_element(row[r], 2), cw_element(row[r], 3)) << 16);
        code[r].y = coded(cw_element(row[r], 4), cw_element(row[r], 5)) | (coded(cw_element(row[r], 6), cw_element(row[r], 7)) << 16);
    }
    if (!is_v) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int i = row0 + r - off;
            const bool fresh = i >= 0 && i < count;
            if (!fresh && off > 0 && !again) continue;    // stays as it is
            reinterpret_cast<uint2*>(data + (row0 + r) * D)[sub] = fresh ? code[r] : off > 0 ? make_uint2(shrunk(old_k[r].x), shrunk(old_k[r].y)) : make_uint2(0u, 0u);
        }
    } else {
        unsigned char* tile = reinterpret_cast<unsigned char*>(sh.tile);
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) tile[(8 * sub + i) * 20 + row0 + r] = (unsigned char)((i < 4 ? code[r].x : code[r].y) >> (8 * (i & 3)));
        __syncthreads();
        if (threadIdx.x < D) {                            // a line of 16 tokens
            unsigned o[4] = {old_v.x, old_v.y, old_v.z, old_v.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                unsigned mask = 0u;
#pragma unroll
                for (int b = 0; b < 4; ++b) mask |= (4 * q + b >= off && 4 * q + b < off + count) ? 0xffu << (8 * b) : 0u;
                if (again) o[q] = shrunk(o[q]);
                o[q] = (sh.tile[threadIdx.x][q] & mask) | (o[q] & ~mask);
            }
            reinterpret_cast<uint4*>(data)[threadIdx.x] = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

template <int D, bool ADJ, bool E4M3, bool QUERIES>
__global__ void __launch_bounds__(CW_WARPS * 32, 6) cache_8bit_write_kernel(const CwParams p) {
    __shared__ CwShared<D> sh;
    static_assert(CW_WARPS * 32 >= D, "a thread for each line of a value block");
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const long long unit = blockIdx.x;
    if (unit >= p.kv_units) {
        if (QUERIES) cw_queries<D, ADJ>(p, (unsigned)(unit - p.kv_units) * CW_WARPS + (threadIdx.x >> 5));
        return;
    }
    const int first = (int)(unit / (2 * p.nkv)) * p.window;
    const int which = (int)(unit % (2 * p.nkv));
    // lane i: token first + i.  A run that begins in the window ends within 15 more tokens.
    const int mine = first + lane;
    const long long slot = mine < p.num_tokens ? p.slot_map[mine] : -1;
    long long before = __shfl_up_sync(0xffffffffu, slot, 1);
    if (lane == 0) before = first > 0 ? p.slot_map[first - 1] : -1;
    const bool there = slot >= 0 && slot < p.num_slots, in_window = lane < p.window && mine < p.num_tokens;
    if (in_window && !there && threadIdx.x < 32) atomicAdd(p.error_count, 1);
    // a token begins a run if the one before it does not lie just before it in the same block
    unsigned begins = __ballot_sync(0xffffffffu, in_window && there && ((slot & (C8_BLOCK - 1)) == 0 || before != slot - 1));
    while (begins != 0u) {                                   // the same in all warps
        const int i = __ffs(begins) - 1;
        begins &= begins - 1;
        const long long start = __shfl_sync(0xffffffffu, slot, i);
        const int room = C8_BLOCK - (int)(start & (C8_BLOCK - 1));
        const unsigned members = __ballot_sync(0xffffffffu, lane >= i && lane < i + room && slot == start + (lane - i)) >> i;
        cw_run<D, ADJ, E4M3>(p, sh, first + i, start, __ffs(~members) - 1, which);
        if (begins != 0u) __syncthreads();
    }
}

template <int D, bool ADJ>
__global__ void __launch_bounds__(CW_WARPS * 32) cache_8bit_queries_kernel(const CwParams p) {
    pdl_wait();
    pdl_trigger();
    cw_queries<D, ADJ>(p, blockIdx.x * CW_WARPS + (threadIdx.x >> 5));
}

template <int D, bool ADJ>
static int cw_launch(const CwParams& p, int code, int* launches, cudaStream_t stream) {
    constexpr int GROUPS = 32 / (D / 8);
    CwParams q = p;
    const bool small = p.num_tokens <= CW_SMALL;
    q.window = small ? 1 : C8_BLOCK;
    q.kv_units = ((long long)p.num_tokens + q.window - 1) / q.window * 2 * p.nkv;
    q.q_shares = max(1, (p.nq + GROUPS * CW_Q_ROWS - 1) / (GROUPS * CW_Q_ROWS));
    const long long q_units = p.nq > 0 ? (long long)p.num_tokens * q.q_shares : 0;
    const long long q_blocks = (q_units + CW_WARPS - 1) / CW_WARPS, kv_blocks = q.kv_units + (small ? q_blocks : 0);
    if (kv_blocks > 2147483647LL || q_units > 2147483647LL) return pi_refuse("pi_cache_8bit_write: %d tokens are beyond the grid limit", p.num_tokens);
    const dim3 threads(CW_WARPS * 32);
    *launches = 1;
    if (!small && q_blocks > 0) {
        pi_launch(cache_8bit_queries_kernel<D, ADJ>, dim3((unsigned)q_blocks), threads, 0, stream, q);
        *launches = 2;
    }
    const dim3 grid((unsigned)kv_blocks);
    if (small) {
        if (code == PI_E4M3) pi_launch(cache_8bit_write_kernel<D, ADJ, true, true>, grid, threads, 0, stream, q);
        else pi_launch(cache_8bit_write_kernel<D, ADJ, false, true>, grid, threads, 0, stream, q);
    } else {
        if (code == PI_E4M3) pi_launch(cache_8bit_write_kernel<D, ADJ, true, false>, grid, threads, 0, stream, q);
        else pi_launch(cache_8bit_write_kernel<D, ADJ, false, false>, grid, threads, 0, stream, q);
    }
    return pi_check_launch("pi_cache_8bit_write");
}

// arguments as one record of 8-byte fields
struct CwArgs {
    const void* qkv; long long row_stride; const void* q_weight; const void* k_weight; long long weight_dtype, has_norm;
    const float* cos_t; const float* sin_t; long long rot_pairs, adjacent;
    void* kcache; void* vcache; float* kscale; float* vscale; long long cache_dtype, num_pages, page_size;
    const long long* slot_map; void* q_out; long long nq, nkv, head_dim, num_tokens; int* error_count;
    double eps;
};

// *launches: kernels launched
PI_EXPORT int pi_cache_8bit_write(const CwArgs* args, int* launches, cudaStream_t stream) {
    const CwArgs& a = *args;
    const int row_stride = (int)a.row_stride, weight_dtype = (int)a.weight_dtype, has_norm = (int)a.has_norm, rot_pairs = (int)a.rot_pairs;
    const int adjacent = (int)a.adjacent, cache_dtype = (int)a.cache_dtype, page_size = (int)a.page_size;
    const int nq = (int)a.nq, nkv = (int)a.nkv, head_dim = (int)a.head_dim, num_tokens = (int)a.num_tokens;
    *launches = 0;
    if (num_tokens <= 0) return 0;
    if (head_dim != 64 && head_dim != 128) return pi_refuse("pi_cache_8bit_write: head size %d is not 64 or 128", head_dim);
    if (nq < 0 || nkv <= 0) return pi_refuse("pi_cache_8bit_write: nq=%d nkv=%d", nq, nkv);
    if (page_size < C8_BLOCK || (page_size & (page_size - 1))) return pi_refuse("pi_cache_8bit_write: page size %d must be a power of two of at least 16", page_size);
    if (cache_dtype != PI_E4M3 && cache_dtype != PI_INT8) return pi_refuse("pi_cache_8bit_write: unknown dtype code %d of the pages", cache_dtype);
    if (has_norm && weight_dtype != PI_F32 && weight_dtype != PI_BF16) return pi_refuse("pi_cache_8bit_write: unknown dtype code %d of the norm weights", weight_dtype);
    if (rot_pairs < 0 || 2 * rot_pairs > head_dim || rot_pairs % (adjacent ? 4 : 8) != 0)
        return pi_refuse("pi_cache_8bit_write: %d rotated pairs must be a multiple of %d and fit the head size %d", rot_pairs, adjacent ? 4 : 8, head_dim);
    if (row_stride % 8 != 0 || row_stride < (nq + 2 * nkv) * head_dim)
        return pi_refuse("pi_cache_8bit_write: rows of %d elements must be a multiple of 8 and hold all heads", row_stride);
    if (((uintptr_t)a.qkv | (uintptr_t)a.q_out | (uintptr_t)a.kcache | (uintptr_t)a.vcache | (uintptr_t)a.cos_t | (uintptr_t)a.sin_t |
         (has_norm ? (uintptr_t)a.q_weight | (uintptr_t)a.k_weight : 0)) & 15)
        return pi_refuse("pi_cache_8bit_write: tensors must start on 16-byte boundaries");
    CwParams p;
    p.qkv = (const bf16*)a.qkv; p.row_stride = row_stride; p.qw = a.q_weight; p.kw = a.k_weight; p.eps = (float)a.eps; p.has_norm = has_norm;
    p.cos_t = a.cos_t; p.sin_t = a.sin_t; p.rot_pairs = rot_pairs;
    p.kcache = (unsigned char*)a.kcache; p.vcache = (unsigned char*)a.vcache; p.kscale = a.kscale; p.vscale = a.vscale;
    p.slot_map = a.slot_map; p.num_slots = a.num_pages * page_size; p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.q_out = (bf16*)a.q_out; p.nq = nq; p.nkv = nkv; p.num_tokens = num_tokens; p.error_count = a.error_count;
    p.kv_units = 0; p.window = p.q_shares = 1; p.wide = weight_dtype == PI_F32;
    if (adjacent)
        return head_dim == 128 ? cw_launch<128, true>(p, cache_dtype, launches, stream) : cw_launch<64, true>(p, cache_dtype, launches, stream);
    return head_dim == 128 ? cw_launch<128, false>(p, cache_dtype, launches, stream) : cw_launch<64, false>(p, cache_dtype, launches, stream);
}

// ---------------------------------------------------------------------------------------------------
// 8-bit pages back to bfloat16: listed page i, tokens [page_tokens[i].x, page_tokens[i].y) (all if page_tokens is null),
// to keys and values [listed][nkv][page_size][D].  Other tokens, and pages outside the pool, become zeros: what reads the
// copies multiplies masked values by zero, so they must be numbers.
// One warp per block of 16 tokens of a head; the values go through shared memory to be turned.
// ---------------------------------------------------------------------------------------------------
#define CR_WARPS 8

struct CrParams {
    const unsigned char* kcache; const unsigned char* vcache; const float* kscale; const float* vscale;
    long long num_pages;
    const int* page_list; const int2* page_tokens; int num_listed;
    bf16* keys; bf16* values;
    int nkv, page_shift;
};

__device__ __forceinline__ unsigned cr_scaled(unsigned half_pair, float scale) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&half_pair));
    const __nv_bfloat162 b = __floats2bfloat162_rn(v.x * scale, v.y * scale);
    return *reinterpret_cast<const unsigned*>(&b);
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(CR_WARPS * 32) cache_8bit_read_kernel(const CrParams p) {
    constexpr int LINE = D + 8;                                // bf16 elements of a token's line in shared memory
    __shared__ __align__(16) bf16 turned[CR_WARPS][C8_BLOCK * LINE];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int page_blocks = 1 << (p.page_shift - 4);
    const long long unit = (long long)blockIdx.x * CR_WARPS + warp;            // (listed page, head, block in the page)
    if (unit >= (long long)p.num_listed * p.nkv * page_blocks) return;
    const int i = (int)(unit / (p.nkv * page_blocks));
    const int rest = (int)(unit - (long long)i * p.nkv * page_blocks);
    const int sub = rest & (page_blocks - 1);
    const int page = p.page_list[i];
    const bool there = page >= 0 && page < p.num_pages;
    int lo = 0, hi = C8_BLOCK;
    if (p.page_tokens != nullptr) {
        const int2 span = p.page_tokens[i];
        lo = span.x - C8_BLOCK * sub; hi = span.y - C8_BLOCK * sub;
    }
    if (!there) hi = lo;
    const long long block = (long long)page * p.nkv * page_blocks + rest;
    const float ks = there ? p.kscale[block] : 0.0f, vs = there ? p.vscale[block] : 0.0f;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    constexpr int PIECES = D / 32;                             // 16-byte pieces of a block per lane
    uint4 k[PIECES], v[PIECES];
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
        k[c] = there ? reinterpret_cast<const uint4*>(p.kcache + (size_t)block * C8_BLOCK * D)[c * 32 + lane] : zero;
        v[c] = there ? reinterpret_cast<const uint4*>(p.vcache + (size_t)block * C8_BLOCK * D)[c * 32 + lane] : zero;
    }
    bf16* kout = p.keys + (size_t)unit * C8_BLOCK * D;         // the copies have the same order of blocks
    bf16* vout = p.values + (size_t)unit * C8_BLOCK * D;
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
        const int piece = c * 32 + lane, tok = piece / (D / 16);
        const bool seen = tok >= lo && tok < hi;
        const unsigned words[4] = {k[c].x, k[c].y, k[c].z, k[c].w};
        unsigned out[8];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            unsigned a, b;
            c8_decode4<E4M3>(words[w], a, b);
            out[2 * w] = seen ? cr_scaled(a, ks) : 0u;
            out[2 * w + 1] = seen ? cr_scaled(b, ks) : 0u;
        }
        uint4* dst = reinterpret_cast<uint4*>(kout + piece * 16);
        dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
        dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
        // a piece of a value block is one line of D: 16 tokens of one element
        const unsigned vw[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
        bf16* column = &turned[warp][piece];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            unsigned a, b;
            c8_decode4<E4M3>(vw[w], a, b);
            const unsigned pair[2] = {cr_scaled(a, vs), cr_scaled(b, vs)};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int tok0 = 4 * w + 2 * h;
                const unsigned short x = tok0 >= lo && tok0 < hi ? (unsigned short)(pair[h] & 0xffffu) : (unsigned short)0;
                const unsigned short y = tok0 + 1 >= lo && tok0 + 1 < hi ? (unsigned short)(pair[h] >> 16) : (unsigned short)0;
                *reinterpret_cast<unsigned short*>(column + tok0 * LINE) = x;
                *reinterpret_cast<unsigned short*>(column + (tok0 + 1) * LINE) = y;
            }
        }
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 2 * PIECES; ++c) {
        const int piece = c * 32 + lane, tok = piece / (D / 8), at = piece % (D / 8);
        reinterpret_cast<uint4*>(vout)[piece] = *reinterpret_cast<const uint4*>(&turned[warp][tok * LINE + at * 8]);
    }
}

struct CrArgs {
    const void* kcache; const void* vcache; const float* kscale; const float* vscale;
    long long cache_dtype, num_pages, nkv, page_size, head_dim;
    const int* page_list; const int* page_tokens; long long num_listed; void* keys; void* values;
};

PI_EXPORT int pi_cache_8bit_read(const CrArgs* args, cudaStream_t stream) {
    const CrArgs& a = *args;
    const int cache_dtype = (int)a.cache_dtype, nkv = (int)a.nkv, page_size = (int)a.page_size, head_dim = (int)a.head_dim;
    const int num_listed = (int)a.num_listed;
    if (num_listed <= 0) return 0;
    if (head_dim != 64 && head_dim != 128) return pi_refuse("pi_cache_8bit_read: head size %d is not 64 or 128", head_dim);
    if (nkv <= 0) return pi_refuse("pi_cache_8bit_read: nkv=%d", nkv);
    if (page_size < C8_BLOCK || (page_size & (page_size - 1))) return pi_refuse("pi_cache_8bit_read: page size %d must be a power of two of at least 16", page_size);
    if (cache_dtype != PI_E4M3 && cache_dtype != PI_INT8) return pi_refuse("pi_cache_8bit_read: unknown dtype code %d of the pages", cache_dtype);
    if (((uintptr_t)a.kcache | (uintptr_t)a.vcache | (uintptr_t)a.keys | (uintptr_t)a.values) & 15)
        return pi_refuse("pi_cache_8bit_read: tensors must start on 16-byte boundaries");
    CrParams p;
    p.kcache = (const unsigned char*)a.kcache; p.vcache = (const unsigned char*)a.vcache; p.kscale = a.kscale; p.vscale = a.vscale;
    p.num_pages = a.num_pages; p.page_list = a.page_list; p.page_tokens = (const int2*)a.page_tokens; p.num_listed = num_listed;
    p.keys = (bf16*)a.keys; p.values = (bf16*)a.values; p.nkv = nkv; p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    const long long units = (long long)num_listed * nkv * (page_size / C8_BLOCK);
    const long long blocks = (units + CR_WARPS - 1) / CR_WARPS;
    if (blocks > 2147483647LL) return pi_refuse("pi_cache_8bit_read: %lld blocks of tokens are beyond the grid limit", units);
    const dim3 grid((unsigned)blocks), threads(CR_WARPS * 32);
    if (head_dim == 128) {
        if (cache_dtype == PI_E4M3) pi_launch(cache_8bit_read_kernel<128, true>, grid, threads, 0, stream, p);
        else pi_launch(cache_8bit_read_kernel<128, false>, grid, threads, 0, stream, p);
    } else {
        if (cache_dtype == PI_E4M3) pi_launch(cache_8bit_read_kernel<64, true>, grid, threads, 0, stream, p);
        else pi_launch(cache_8bit_read_kernel<64, false>, grid, threads, 0, stream, p);
    }
    return pi_check_launch("pi_cache_8bit_read");
}
