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
// One warp per (run, kv head, key or value): the scale needs the whole run, and a run is at most 16 rows of D elements -
// 4 KB, held in registers.  Lanes of D / 8 form a group that takes 16-byte pieces of a row; a group takes consecutive
// rows, so that for values its lanes hold consecutive bytes of the transposed block.  The warp of a token that does not
// begin a run ends at once.  Query heads are plain streaming work, two rows in flight per group.
// ---------------------------------------------------------------------------------------------------
#define CW_WARPS 8
#define CW_Q_ROWS 2          // query rows in flight per lane group

struct CwParams {
    const bf16* qkv; int row_stride;
    const void* qw; const void* kw; float eps; int has_norm;
    const float* cos_t; const float* sin_t; int rot_pairs, adjacent;
    unsigned char* kcache; unsigned char* vcache; float* kscale; float* vscale;
    const long long* slot_map; long long num_slots; int page_shift;
    bf16* q_out;
    int nq, nkv, num_tokens;
    long long kv_units, q_units;      // warps' worth of work
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
template <typename TW>
__device__ __forceinline__ void cw_weights(const void* w, int sub, float (&v)[8]) {
    if constexpr (sizeof(TW) == 2) {
        cw_unpack(reinterpret_cast<const uint4*>(w)[sub], v);
    } else {
        const float4 a = reinterpret_cast<const float4*>(w)[2 * sub], b = reinterpret_cast<const float4*>(w)[2 * sub + 1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
}

// norm and rotation of one row spread over D / 8 lanes; every lane of the warp calls it (x of rows that do not exist: zeros)
template <int D>
__device__ __forceinline__ void cw_norm_rope(const CwParams& p, int t, int sub, const float (&w)[8], float (&x)[8]) {
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
    const size_t row = (size_t)t * p.rot_pairs;
    if (p.adjacent) {                                   // pairs (2i, 2i + 1); rot_pairs is a multiple of 4
        if (4 * sub < p.rot_pairs) {
            const float4 c = *reinterpret_cast<const float4*>(p.cos_t + row + 4 * sub);
            const float4 s = *reinterpret_cast<const float4*>(p.sin_t + row + 4 * sub);
            const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const float r0 = x[2 * h] * cs[h] - x[2 * h + 1] * sn[h], r1 = x[2 * h] * sn[h] + x[2 * h + 1] * cs[h];
                x[2 * h] = r0; x[2 * h + 1] = r1;
            }
        }
    } else {                                            // pairs (i, i + rot_pairs); rot_pairs is a multiple of 8
        const int shift = p.rot_pairs / 8;              // the partner's lane
        const bool first = sub < shift, second = !first && sub < 2 * shift;
        const int partner = first ? sub + shift : second ? sub - shift : sub;
        float other[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xffffffffu, x[i], partner, LANES);
        if (first || second) {
            const int at = 8 * (first ? sub : sub - shift);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float4 c = *reinterpret_cast<const float4*>(p.cos_t + row + at + 4 * q);
                const float4 s = *reinterpret_cast<const float4*>(p.sin_t + row + at + 4 * q);
                const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const int i = 4 * q + h;
                    x[i] = first ? x[i] * cs[h] - other[i] * sn[h] : other[i] * sn[h] + x[i] * cs[h];
                }
            }
        }
    }
}

// element i (0..7) of four registers of bf16 pairs
__device__ __forceinline__ float cw_element(const uint4& raw, int i) {
    const unsigned w = i < 2 ? raw.x : i < 4 ? raw.y : i < 6 ? raw.z : raw.w;
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
}

template <int D, typename TW, bool E4M3>
__global__ void __launch_bounds__(CW_WARPS * 32) cache_8bit_write_kernel(const CwParams p) {
    constexpr int LANES = D / 8, GROUPS = 32 / LANES, ROWS = C8_BLOCK / GROUPS;       // D 128: 2 groups of 8 rows; 64: 4 of 4
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, sub = lane % LANES, grp = lane / LANES;
    const long long unit = (long long)blockIdx.x * CW_WARPS + (threadIdx.x >> 5);
    if (unit >= p.kv_units) {
        // ---- query rows: (token, head) pairs ------------------------------------------------------------------
        const long long q_unit = unit - p.kv_units;
        if (q_unit >= p.q_units) return;
        float w[8];
        if (p.has_norm) cw_weights<TW>(p.qw, sub, w);
        uint4 raw[CW_Q_ROWS];
        int tok[CW_Q_ROWS], head[CW_Q_ROWS];
        const long long rows = (long long)p.num_tokens * p.nq;
#pragma unroll
        for (int j = 0; j < CW_Q_ROWS; ++j) {
            const long long row = (q_unit * CW_Q_ROWS + j) * GROUPS + grp;
            tok[j] = row < rows ? (int)(row / p.nq) : -1;
            head[j] = row < rows ? (int)(row - (long long)tok[j] * p.nq) : 0;
            raw[j] = tok[j] >= 0 ? reinterpret_cast<const uint4*>(p.qkv + (size_t)tok[j] * p.row_stride + head[j] * D)[sub]
                                 : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int j = 0; j < CW_Q_ROWS; ++j) {
            float x[8];
            cw_unpack(raw[j], x);
            cw_norm_rope<D>(p, max(tok[j], 0), sub, w, x);
            if (tok[j] >= 0) reinterpret_cast<uint4*>(p.q_out + ((size_t)tok[j] * p.nq + head[j]) * D)[sub] = cw_pack(x);
        }
        return;
    }
    // ---- a run of tokens in one block of one key or value head ----------------------------------------------------
    const int t = (int)(unit / (2 * p.nkv));
    const int which = (int)(unit - (long long)t * 2 * p.nkv);
    const bool is_v = which >= p.nkv;
    const int head = is_v ? which - p.nkv : which;
    const long long slot = p.slot_map[t];
    if (slot < 0 || slot >= p.num_slots) {
        if (lane == 0) atomicAdd(p.error_count, 1);
        return;
    }
    const int off = (int)(slot & (C8_BLOCK - 1));
    if (off != 0 && t > 0 && p.slot_map[t - 1] == slot - 1) return;                    // its run began earlier
    int count;
    {
        const bool member = lane < C8_BLOCK - off && t + lane < p.num_tokens && p.slot_map[t + lane] == slot + lane;
        count = __ffs(~__ballot_sync(0xffffffffu, member)) - 1;                        // at least 1
    }
    const int page_blocks = 1 << (p.page_shift - 4);
    const long long page = slot >> p.page_shift;
    const long long block = (page * p.nkv + head) * page_blocks + (((int)slot & ((1 << p.page_shift) - 1)) >> 4);
    unsigned char* data = (is_v ? p.vcache : p.kcache) + (size_t)block * C8_BLOCK * D;
    float* scale = (is_v ? p.vscale : p.kscale) + block;

    // the new rows, in bf16, and their largest magnitude
    const bf16* src = p.qkv + (size_t)t * p.row_stride + (size_t)(p.nq + which) * D;
    uint4 row[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int i = grp * ROWS + r - off;                                             // token t + i
        row[r] = (i >= 0 && i < count) ? reinterpret_cast<const uint4*>(src + (size_t)i * p.row_stride)[sub] : make_uint4(0u, 0u, 0u, 0u);
    }
    if (!is_v) {
        float w[8];
        if (p.has_norm) cw_weights<TW>(p.kw, sub, w);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int i = grp * ROWS + r - off;
            float x[8];
            cw_unpack(row[r], x);
            cw_norm_rope<D>(p, t + max(0, min(i, count - 1)), sub, w, x);
            if (i >= 0 && i < count) row[r] = cw_pack(x);
        }
    }
    float amax = 0.0f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(cw_element(row[r], i)));     // fmaxf passes over NaN
    }
    amax = warp_max(amax);
    int e = c8_exponent<E4M3>(amax), e_old = e;
    if (off > 0) { e_old = c8_scale_exponent(*scale); e = max(e, e_old); }
    const bool again = off > 0 && e != e_old;             // what lies in the block is encoded again
    const float inv = c8_pow2(-e), shrink = c8_pow2(e_old - e);
    __syncwarp();
    if (lane == 0 && (off == 0 || again)) *scale = c8_pow2(e);
    auto coded = [&](float a, float b) -> unsigned {
        a = a == a ? a * inv : 0.0f;
        b = b == b ? b * inv : 0.0f;
        return c8_encode2<E4M3>(a, b);
    };
    auto shrunk = [&](unsigned codes) -> unsigned {       // two old codes at the new scale
        const float2 v = __half22float2(c8_decode2<E4M3>(codes));
        return c8_encode2<E4M3>(v.x * shrink, v.y * shrink);
    };
    if (!is_v) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int at = grp * ROWS + r, i = at - off;
            const bool fresh = i >= 0 && i < count;
            if (!fresh && off > 0 && !again) continue;
            uint2* dst = reinterpret_cast<uint2*>(data + at * D) + sub;
            uint2 out = make_uint2(0u, 0u);
            if (fresh) {
                out.x = coded(cw_element(row[r], 0), cw_element(row[r], 1)) | (coded(cw_element(row[r], 2), cw_element(row[r], 3)) << 16);
                out.y = coded(cw_element(row[r], 4), cw_element(row[r], 5)) | (coded(cw_element(row[r], 6), cw_element(row[r], 7)) << 16);
            } else if (off > 0) {
                const uint2 old = *dst;
                out.x = shrunk(old.x & 0xffffu) | (shrunk(old.x >> 16) << 16);
                out.y = shrunk(old.y & 0xffffu) | (shrunk(old.y >> 16) << 16);
            }
            *dst = out;
        }
    } else {
        // element i of the lane's rows: ROWS consecutive bytes of line 8 sub + i of the transposed block
        const int lo = grp * ROWS - off;                  // token (counted from t) of the lane's first row
        const bool any_fresh = lo < count && lo + ROWS > 0;
        if (!any_fresh && off > 0 && !again) return;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            unsigned* dst = reinterpret_cast<unsigned*>(data + (8 * sub + i) * C8_BLOCK + grp * ROWS);
#pragma unroll
            for (int q = 0; q < ROWS / 4; ++q) {
                unsigned old = 0u;
                if (off > 0) {
                    old = dst[q];
                    if (again) old = shrunk(old & 0xffffu) | (shrunk(old >> 16) << 16);
                }
                const unsigned fresh = coded(cw_element(row[4 * q], i), cw_element(row[4 * q + 1], i)) |
                                       (coded(cw_element(row[4 * q + 2], i), cw_element(row[4 * q + 3], i)) << 16);
                unsigned mask = 0u;
#pragma unroll
                for (int b = 0; b < 4; ++b) mask |= (lo + 4 * q + b >= 0 && lo + 4 * q + b < count) ? 0xffu << (8 * b) : 0u;
                dst[q] = (fresh & mask) | (old & ~mask);
            }
        }
    }
}

template <int D>
static int cw_launch(const CwParams& p, int weight_dtype, int code, cudaStream_t stream) {
    constexpr int GROUPS = 32 / (D / 8);
    CwParams q = p;
    q.kv_units = (long long)p.num_tokens * 2 * p.nkv;
    q.q_units = ((long long)p.num_tokens * p.nq + GROUPS * CW_Q_ROWS - 1) / (GROUPS * CW_Q_ROWS);
    const long long blocks = (q.kv_units + q.q_units + CW_WARPS - 1) / CW_WARPS;
    if (blocks > 2147483647LL) return pi_refuse("pi_cache_8bit_write: %d tokens are beyond the grid limit", p.num_tokens);
    const dim3 grid((unsigned)blocks), threads(CW_WARPS * 32);
    const bool wide = weight_dtype == PI_F32;
    if (code == PI_E4M3) {
        if (wide) pi_launch(cache_8bit_write_kernel<D, float, true>, grid, threads, 0, stream, q);
        else pi_launch(cache_8bit_write_kernel<D, bf16, true>, grid, threads, 0, stream, q);
    } else {
        if (wide) pi_launch(cache_8bit_write_kernel<D, float, false>, grid, threads, 0, stream, q);
        else pi_launch(cache_8bit_write_kernel<D, bf16, false>, grid, threads, 0, stream, q);
    }
    return pi_check_launch("pi_cache_8bit_write");
}

PI_EXPORT int pi_cache_8bit_write(const void* qkv, int row_stride, const void* q_weight, const void* k_weight, int weight_dtype,
                                  float eps, int has_norm, const float* cos_t, const float* sin_t, int rot_pairs, int adjacent,
                                  void* kcache, void* vcache, float* kscale, float* vscale, int cache_dtype, long long num_pages,
                                  int page_size, const long long* slot_map, void* q_out, int nq, int nkv, int head_dim,
                                  int num_tokens, int* error_count, cudaStream_t stream) {
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
    if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)cos_t | (uintptr_t)sin_t |
         (has_norm ? (uintptr_t)q_weight | (uintptr_t)k_weight : 0)) & 15)
        return pi_refuse("pi_cache_8bit_write: tensors must start on 16-byte boundaries");
    CwParams p;
    p.qkv = (const bf16*)qkv; p.row_stride = row_stride; p.qw = q_weight; p.kw = k_weight; p.eps = eps; p.has_norm = has_norm;
    p.cos_t = cos_t; p.sin_t = sin_t; p.rot_pairs = rot_pairs; p.adjacent = adjacent;
    p.kcache = (unsigned char*)kcache; p.vcache = (unsigned char*)vcache; p.kscale = kscale; p.vscale = vscale;
    p.slot_map = slot_map; p.num_slots = num_pages * page_size; p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.q_out = (bf16*)q_out; p.nq = nq; p.nkv = nkv; p.num_tokens = num_tokens; p.error_count = error_count;
    p.kv_units = p.q_units = 0;
    return head_dim == 128 ? cw_launch<128>(p, weight_dtype, cache_dtype, stream) : cw_launch<64>(p, weight_dtype, cache_dtype, stream);
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

PI_EXPORT int pi_cache_8bit_read(const void* kcache, const void* vcache, const float* kscale, const float* vscale, int cache_dtype,
                                 long long num_pages, int nkv, int page_size, int head_dim, const int* page_list,
                                 const int* page_tokens, int num_listed, void* keys, void* values, cudaStream_t stream) {
    if (num_listed <= 0) return 0;
    if (head_dim != 64 && head_dim != 128) return pi_refuse("pi_cache_8bit_read: head size %d is not 64 or 128", head_dim);
    if (nkv <= 0) return pi_refuse("pi_cache_8bit_read: nkv=%d", nkv);
    if (page_size < C8_BLOCK || (page_size & (page_size - 1))) return pi_refuse("pi_cache_8bit_read: page size %d must be a power of two of at least 16", page_size);
    if (cache_dtype != PI_E4M3 && cache_dtype != PI_INT8) return pi_refuse("pi_cache_8bit_read: unknown dtype code %d of the pages", cache_dtype);
    if (((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)keys | (uintptr_t)values) & 15)
        return pi_refuse("pi_cache_8bit_read: tensors must start on 16-byte boundaries");
    CrParams p;
    p.kcache = (const unsigned char*)kcache; p.vcache = (const unsigned char*)vcache; p.kscale = kscale; p.vscale = vscale;
    p.num_pages = num_pages; p.page_list = page_list; p.page_tokens = (const int2*)page_tokens; p.num_listed = num_listed;
    p.keys = (bf16*)keys; p.values = (bf16*)values; p.nkv = nkv; p.page_shift = 0;
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
