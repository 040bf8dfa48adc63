// Decode attention over 8-bit key/value pages (format: cache_8bit.cuh): segments of one token,
//   out = softmax(scale * q K^T) V,  K = 2^ek k8,  V = 2^ev v8,  keys lo .. pos (lo = pos - window + 1 with a window)
//
// All of it is memory traffic - each byte of a key or value is used for a handful of query heads - so keys and values go
// straight from memory into the registers in which mma.sync wants them, in 16-byte pieces, and nothing is exchanged between
// warps until all work is done.  A warp takes 64 keys (four blocks of 16) at a time: while it computes the scores of a tile
// its values are on their way, and as soon as a register of keys or values has been used, the next tile's is asked for: 8 to
// 16 KB per warp, about 100 KB per SM, in flight.
//   S^T = K Q^T      m16n8k16, 16 keys x 8 query heads; the codes become half precision exactly (two instructions for four
//                    e4m3, five for int8), queries are scaled to [1, 2) per head so that half precision holds them
//   softmax          in 32 bits; a value block's scale joins the exponent: w = 2^(s + ev - m'), m' the running maximum of
//                    s + ev, so the weights of the second product are at most 1 whatever the scales are (half precision
//                    rounds them by up to 2^-11), and the sum of 2^(s - m') is kept beside it
//   O^T += V^T w^T   m16n8k16, 16 elements of the head x 8 query heads; movmatrix turns the weights, and V^T is what the
//                    pages hold
// The contractions do not care in which order keys or elements come, so the order is the one in which a lane's pieces lie:
//   keys     tile of 16 rows j = 0..3: row r holds token 4 j + (r & 1) + 2 (r >> 3) of block (r & 7) >> 1
//   elements lane t of a quad holds elements 64 c + 16 t .. + 15 of its rows, four of them per k step
//   tokens   lane t of a quad holds block t of each line of V^T, four tokens per k step j: those of the keys' tile j
//
// Work split: the 64-key tiles of all (request, kv head, eight query heads) triples form one sequence, `pair_cost` units
// before each; every CTA (one per SM) takes an equal share of it and every warp an equal share of its CTA's, whatever the
// lengths of the requests.  A warp runs through its pieces without waiting for another warp, asking ahead across the
// boundaries of pieces.  A triple inside one warp's share is written by that warp.  The others are added up through shared
// memory, once, when all warps are done; what was cut between CTAs leaves (maximum, sum, accumulator) in the workspace, and the
// CTA that delivers a triple's last missing piece adds the pieces up in the order of the keys.  Nothing waits for another CTA.
// A group of more than eight query heads is cut in pieces of eight, and its keys are read once for each (from L2 mostly).
//
// Measured (B200, 8 kv heads of 128; device time of a launch among others): 64 requests of 130 to 8,190 keys, 40 query heads,
// e4m3: 85 us, 459 MB at 5.4 TB/s (6.9 in the middle); 8 requests of 4,096 keys: 21.4 us for
// 10.2 us of transfer: the first tiles are asked for after 2.5 to 4.5 us (lengths, block table), by all SMs at once, and are
// there after 6.5 to 9; a warp has three or four tiles and is done after 8 to 19; the sums between warps and CTAs take 3.  One
// request of 32,768 keys, int8: 23.4 us.  Tried: operands through a queue in shared memory of each warp, by bulk copies with an mbarrier per
// 4 KB (83, 22.7 and 25.4 us; also with 12 warps) or by cp.async (slower still); spans of whole CTAs, a barrier at each piece
// (113, 25.8 and 31.7 us); shares counted in blocks of 16 keys instead of tiles of 64 (evener, but more cuts and tiles that are
// not full: 85.2, 21.7 and 24.3 us).
// The shortest share of a CTA (span_min) is two units and pair_cost two: one to four units a CTA are alike within 0.3 us for 1 to 16
// requests of up to 700 keys (8.4 to 11.5 us; 8 units: 0.5 to 1.2 us slower, 16: 2 to 4.4 us, though three requests behind a window
// of 130 take 7.4 instead of 8.4), no cost at all 0.4 us slower for 8 x 4,096 keys and for 32,768, a cost of four 1 to 2 us slower
// for 16 to 64 requests.
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

// what the kernel needs of the segments, in shared memory
struct A8Meta {
    int pre[A8_MAX_SEGS + 1];       // first unit of a segment; pre[num_segments]: their number
    int pos[A8_MAX_SEGS], slot[A8_MAX_SEGS], row[A8_MAX_SEGS];
};

struct A8Piece {
    int seg, slot, kvh, h0, heads, pos, lo, tile, ntiles;   // tile: first 64-key tile of the piece (absolute)
    int unit0, tiles;                                  // unit of the triple's first tile, and how many tiles the triple has
    int begins, ends;                                  // the piece holds the triple's first / last tile
};

struct A8Cursor { int f, end, seg; };

// n units in equal shares
struct A8Shares {
    int each, more;                 // the first `more` shares have each + 1 units
    __device__ __forceinline__ A8Shares(int n, int shares) : each(n / shares), more(n - n / shares * shares) {}
    __device__ __forceinline__ int from(int share) const { return share * each + min(share, more); }
    __device__ __forceinline__ int holds(int unit) const {      // the share of a unit
        const int longer = more * (each + 1);
        return unit < longer ? unit / (each + 1) : more + (unit - longer) / each;
    }
};

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

__device__ __forceinline__ int a8_lo(const A8Params& p, int pos) { return p.window > 0 ? max(0, pos - p.window + 1) : 0; }

// a cursor over the units [from, to) of the sequence
__device__ __forceinline__ void a8_begin(const A8Params& p, const A8Meta& meta, int from, int to, A8Cursor& c) {
    c.f = from;
    c.end = to;
    int lo = 0, hi = p.num_segments;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (meta.pre[mid] <= from) lo = mid; else hi = mid;
    }
    c.seg = lo;
}

__device__ __forceinline__ bool a8_next(const A8Params& p, const A8Meta& meta, A8Cursor& c, A8Piece& w) {
    if (c.f >= c.end) return false;
    while (meta.pre[c.seg + 1] <= c.f) ++c.seg;                       // ends: f lies before the end of the sequence
    const int first = meta.pre[c.seg];
    w.pos = meta.pos[c.seg];
    w.lo = a8_lo(p, w.pos);
    const int n = w.pos / A8_TILE - w.lo / A8_TILE + 1, per = n + p.pair_cost;
    const int triple = (c.f - first) / per;
    const int unit0 = first + triple * per + p.pair_cost;             // unit of the triple's first tile
    const int lo_u = max(c.f, unit0), hi_u = min(c.end, unit0 + n);
    c.f = hi_u;
    if (hi_u <= lo_u) { c.f = c.end; return false; }                  // the span ends among the cost units
    w.kvh = p.head_tiles == 1 ? triple : triple / p.head_tiles;
    const int ht = triple - w.kvh * p.head_tiles;
    w.seg = c.seg;
    w.slot = meta.slot[c.seg];
    w.h0 = w.kvh * p.group + ht * A8_HEADS;
    w.heads = min(A8_HEADS, p.group - ht * A8_HEADS);
    w.tile = w.lo / A8_TILE + (lo_u - unit0);
    w.ntiles = hi_u - lo_u;
    w.unit0 = unit0; w.tiles = n;
    w.begins = lo_u == unit0; w.ends = hi_u == unit0 + n;
    return true;
}

// four elements of the result, at `at` in the output
__device__ __forceinline__ void a8_write4(const A8Params& p, int row, size_t at, const float4& sum, float den) {
    if (row < 0 || row >= p.num_tokens) return;
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
    const __nv_bfloat162 a = __floats2bfloat162_rn(sum.x * inv, sum.y * inv), b = __floats2bfloat162_rn(sum.z * inv, sum.w * inv);
    *reinterpret_cast<uint2*>(p.out + at) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

// a triple that was cut between warps or CTAs
struct A8Join {
    int first, which, stop;         // the CTA's warps that hold parts of it; the first one's lies in its slot `which`
    int whole;                      // all of it lies in this CTA
    int h0, heads, row;
    int cta0, pieces;               // otherwise: the CTA it begins in, and how many it reaches into
};

// what a block keeps in shared memory
template <int D>
struct A8Shared {
    static constexpr int LINE = D + 4;                    // floats of a head's line: no bank conflicts
    float parts[A8_WARPS * 2][A8_HEADS][LINE];            // per warp: of the triple that began before its span, and of one that begins in it
    float m[A8_WARPS * 2][A8_HEADS], l[A8_WARPS * 2][A8_HEADS];
    A8Meta meta;
    int scan[32];
    A8Join join[A8_WARPS + 1];
    int joins;                                            // of those that begin in the CTA
    int cut[2];                                           // which join left its sum in workspace slot 0 and 1; -1: none
    int last[2];

    __device__ __forceinline__ float* part(int warp, int which, int head) { return parts[2 * warp + which][head]; }
};

template <int D, bool E4M3>
__global__ void __launch_bounds__(A8_THREADS, 1) attn_decode_8bit_kernel(const A8Params p) {
    typedef A8Shared<D> Shared;
    constexpr int KC = D / 64;             // 16-byte pieces of a key row per lane
    constexpr int KS = D / 16;             // k steps of the first product, and 16-row tiles of V^T
    extern __shared__ __align__(16) unsigned char a8_smem[];
    Shared& sh = *reinterpret_cast<Shared*>(a8_smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const A8Meta& meta = sh.meta;
    if (threadIdx.x < 2) sh.cut[threadIdx.x] = -1;
    if (threadIdx.x == 0) { sh.joins = 0; sh.join[0].heads = 0; }
    if (threadIdx.x < A8_WARPS * 2 * A8_HEADS) { (&sh.m[0][0])[threadIdx.x] = -INFINITY; (&sh.l[0][0])[threadIdx.x] = 0.0f; }
    static_assert(A8_WARPS * 2 * A8_HEADS <= A8_THREADS, "one thread per entry");
    pdl_wait();
    const int page_blocks = 1 << (p.page_shift - 4);
    {   // the segments' units, summed up by the whole block
        const int triples = p.nkv * p.head_tiles;
        const long long most = ((long long)p.bt_stride << p.page_shift) - 1;         // a position is kept within the block table
        int run = 0;
        for (int s0 = 0; s0 < p.num_segments; s0 += A8_THREADS) {
            const int s = s0 + threadIdx.x;
            int n = 0;
            if (s < p.num_segments) {
                const int len = p.seg_len[s], start = p.seg_start[s], slot = p.seg_slot[s], row = p.seg_off[s];
                const int pos = (int)min((long long)start, most);
                if (len == 1 && pos >= 0) n = triples * (pos / A8_TILE - a8_lo(p, pos) / A8_TILE + 1 + p.pair_cost);
                sh.meta.pos[s] = pos; sh.meta.slot[s] = slot; sh.meta.row[s] = row;
            }
            int inc = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += a;
            }
            if (lane == 31) sh.scan[warp] = inc;
            __syncthreads();
            int before = run;
#pragma unroll
            for (int x = 0; x < A8_WARPS; ++x) {
                const int sum = sh.scan[x];
                if (x < warp) before += sum;
                run += sum;
            }
            if (s < p.num_segments) sh.meta.pre[s] = before + inc - n;
            if (s0 + A8_THREADS < p.num_segments) __syncthreads();
        }
        if (threadIdx.x == 0) sh.meta.pre[p.num_segments] = run;
    }
    __syncthreads();
    // equal shares of all units for the CTAs (the first ones have one more where it does not come out even), and of a CTA's
    // units for its warps
    const int total = meta.pre[p.num_segments];
    const int ctas = min((int)gridDim.x, (total + p.span_min - 1) / p.span_min);
    if ((int)blockIdx.x >= ctas) return;
    const A8Shares of_ctas(total, ctas);
    const int cta_from = of_ctas.from(blockIdx.x), cta_len = of_ctas.from(blockIdx.x + 1) - cta_from;
    const A8Shares of_warps(cta_len, A8_WARPS);

    // block (lane >> 3) of a tile of piece x: its number in the pool, -1 if it holds no visible key or has no page
    auto lookup = [&](const A8Piece& x, int tile) -> int {
        const int key = tile * A8_TILE + (lane >> 3) * C8_BLOCK;
        if (x.slot < 0 || x.slot >= p.bt_rows || key > x.pos || key + C8_BLOCK <= x.lo) return -1;
        const int page = p.block_table[(size_t)x.slot * p.bt_stride + (key >> p.page_shift)];
        if (page < 0 || page >= p.num_pages) return -1;
        return (page * p.nkv + x.kvh) * page_blocks + ((key & ((1 << p.page_shift) - 1)) >> 4);
    };
    uint4 kr[4][2][KC], vr[KS][2];
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
    A8Cursor cur;
    a8_begin(p, meta, cta_from + of_warps.from(warp), cta_from + of_warps.from(warp + 1), cur);
    A8Piece w, following;
    bool valid = a8_next(p, meta, cur, w);
    int id = 0;
    float ks = 0.0f, vs = 0.0f;
    if (valid) {
        id = lookup(w, w.tile);
        load_k(id);
        load_v(__shfl_sync(0xffffffffu, id, 8 * t));
        ks = p.kscale[max(id, 0)]; vs = p.vscale[max(id, 0)];
    }
    while (valid) {
        const bool have_next = a8_next(p, meta, cur, following);
        const int row = meta.row[w.seg];
        // queries of head g as the second operand, scaled by a power of two into [1, 2); lanes of heads that are not: zeros
        unsigned qb[KS][2];
        float f0, f1;
        {
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
        for (int left = w.ntiles, tile = w.tile; left > 0; --left, ++tile) {
            const bool more = left > 1 || have_next;
            const int id_next = left > 1 ? lookup(w, tile + 1) : have_next ? lookup(following, following.tile) : -1;
            float ks_next = 0.0f, vs_next = 0.0f;
            float s[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { s[j][0] = 0.0f; s[j][1] = 0.0f; s[j][2] = 0.0f; s[j][3] = 0.0f; }
#pragma unroll
            for (int k = 0; k < KS; ++k) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
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
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int m = 0; m < KS; ++m) {
                    unsigned a0, a1, a2, a3;
                    c8_decode4<E4M3>(a8_word(vr[m][0], j), a0, a2);
                    c8_decode4<E4M3>(a8_word(vr[m][1], j), a1, a3);
                    a8_mma(o[m], a0, a1, a2, a3, pb[j][0], pb[j][1]);
                }
            }
            if (more) load_v(__shfl_sync(0xffffffffu, id_next, 8 * t));
            id = id_next; ks = ks_next; vs = vs_next;
        }
        // ---- the end of the piece -----------------------------------------------------------------------------------------
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) { l0 += __shfl_xor_sync(0xffffffffu, l0, d); l1 += __shfl_xor_sync(0xffffffffu, l1, d); }
        if (w.begins && w.ends) {                         // the whole triple
            const float i0 = l0 == 0.0f ? 0.0f : 1.0f / l0, i1 = l1 == 0.0f ? 0.0f : 1.0f / l1;
            const bool odd = (g & 1) != 0;                // lanes of neighbouring elements: the even one takes head 2t, the odd one 2t + 1
            const int head = 2 * t + (odd ? 1 : 0);
            bf16* dst = p.out + ((size_t)max(row, 0) * p.nq + w.h0 + head) * D + (g & ~1);
            const bool write = row >= 0 && row < p.num_tokens && head < w.heads;
#pragma unroll
            for (int m = 0; m < KS; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float a = o[m][2 * h] * i0, b = o[m][2 * h + 1] * i1;
                    const float got = __shfl_xor_sync(0xffffffffu, odd ? a : b, 4);
                    const __nv_bfloat162 v = odd ? __floats2bfloat162_rn(got, b) : __floats2bfloat162_rn(a, got);
                    if (write) *reinterpret_cast<__nv_bfloat162*>(dst + 16 * m + 8 * h) = v;
                }
        } else {                                          // a part of one; one that begins here is the span's last piece
            const int unit = w.unit0 + w.tile - w.lo / A8_TILE, last_unit = w.unit0 + w.tiles - 1;
            if (lane == 0 && (w.begins || unit == cta_from)) {      // the triple's first part in this CTA: noted for the sum below
                const int at = w.begins ? atomicAdd(&sh.joins, 1) + 1 : 0;
                A8Join& j = sh.join[at];
                j.first = warp; j.which = w.begins;
                j.stop = last_unit < cta_from + cta_len ? of_warps.holds(last_unit - cta_from) : A8_WARPS - 1;
                j.whole = w.begins && last_unit < cta_from + cta_len;
                j.h0 = w.h0; j.heads = w.heads; j.row = row;
                if (!j.whole) {
                    j.cta0 = w.begins ? blockIdx.x : of_ctas.holds(w.unit0);
                    j.pieces = of_ctas.holds(last_unit) - j.cta0 + 1;
                }
            }
            const int part = warp * 2 + w.begins;
            if (g == 0) {
                sh.m[part][2 * t] = m0; sh.m[part][2 * t + 1] = m1;
                sh.l[part][2 * t] = l0; sh.l[part][2 * t + 1] = l1;
            }
            float* p0 = sh.part(warp, w.begins, 2 * t);
            float* p1 = sh.part(warp, w.begins, 2 * t + 1);
#pragma unroll
            for (int m = 0; m < KS; ++m) {
                p0[16 * m + g] = o[m][0]; p1[16 * m + g] = o[m][1];
                p0[16 * m + 8 + g] = o[m][2]; p1[16 * m + 8 + g] = o[m][3];
            }
        }
        valid = have_next;
        w = following;
    }
    // (The next kernel is not let in early: with a pdl_trigger() here the product behind this
    // kernel spreads unevenly over the SMs that end first, and a decode step of 36 layers goes from 3.9 to 6.3 ms.)
    __syncthreads();
    // ---- triples that were cut between the warps of the CTA: their parts are added up in warp order.  Join 0 is a triple that
    // began before the CTA, at most one of the others goes on behind it; these two leave their sum in the workspace -----------
    const int joins = sh.joins + 1;
    const int team = joins > A8_WARPS / 2 ? 1 : A8_WARPS / joins;                     // warps per triple
    for (int at = warp / team; at < joins; at += A8_WARPS / team) {
        const A8Join& j = sh.join[at];
        if (j.heads == 0) continue;
        for (int i = (warp % team) * 32 + lane; i < j.heads * (D / 4); i += team * 32) {
            const int h = i / (D / 4), e = 4 * (i % (D / 4));
            float f[A8_WARPS], top = -INFINITY, den = 0.0f;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            bool has[A8_WARPS];                               // a warp with an empty span, or without a visible key, has no part
#pragma unroll
            for (int x = 0; x < A8_WARPS; ++x) {
                const int part = 2 * x + (x == j.first ? j.which : 0);
                has[x] = x >= j.first && x <= j.stop && !(sh.m[part][h] == -INFINITY && sh.l[part][h] == 0.0f);
                f[x] = has[x] ? sh.m[part][h] : -INFINITY;
                top = fmaxf(top, f[x]);
            }
            const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int x = 0; x < A8_WARPS; ++x) {
                if (!has[x]) continue;
                const int which = x == j.first ? j.which : 0;
                const float wgt = a8_ex2(f[x] - ref);
                const float4 v = *reinterpret_cast<const float4*>(sh.part(x, which, h) + e);
                sum.x = fmaf(wgt, v.x, sum.x); sum.y = fmaf(wgt, v.y, sum.y); sum.z = fmaf(wgt, v.z, sum.z); sum.w = fmaf(wgt, v.w, sum.w);
                den = fmaf(wgt, sh.l[2 * x + which][h], den);
            }
            if (j.whole) {
                a8_write4(p, j.row, ((size_t)j.row * p.nq + j.h0 + h) * D + e, sum, den);
            } else {
                const size_t to = ((size_t)blockIdx.x * 2 + j.which) * A8_SLOT_HEADS + h;
                *reinterpret_cast<float4*>(p.ws_acc + to * D + e) = sum;
                if (e == 0) *reinterpret_cast<float2*>(p.ws_ml + to * 2) = make_float2(top, den);
            }
        }
        if (!j.whole && lane == 0 && warp % team == 0) sh.cut[j.which] = at;
    }
    // ---- triples that were cut between CTAs: the CTA that delivers the last piece adds them up in the order of the keys ------
    __syncthreads();
    if (threadIdx.x < 2) {
        int last = 0;
        if (sh.cut[threadIdx.x] >= 0) {
            const A8Join& j = sh.join[sh.cut[threadIdx.x]];
            __threadfence();                                  // the whole block's writes (the barrier above) before the count
            last = atomicAdd(&p.ws_count[j.cta0], 1u) + 1 == (unsigned)j.pieces;
            if (last) p.ws_count[j.cta0] = 0u;                // zero for the next launch
            __threadfence();
        }
        sh.last[threadIdx.x] = last;
    }
    __syncthreads();
    constexpr int HALF_BLOCK = A8_THREADS / 2;                // one half of the block for each of the two
    const int c = threadIdx.x / HALF_BLOCK;
    if (!sh.last[c]) return;
    const A8Join& j = sh.join[sh.cut[c]];
    for (int i = threadIdx.x % HALF_BLOCK; i < j.heads * (D / 4); i += HALF_BLOCK) {
        const int h = i / (D / 4), e = 4 * (i % (D / 4));
        float top = -INFINITY, den = 0.0f;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        constexpr int BATCH = 10;                             // pieces whose loads are in flight together
        for (int x0 = 0; x0 < j.pieces; x0 += BATCH) {
            float2 ml[BATCH];
            float4 v[BATCH];
#pragma unroll
            for (int x = 0; x < BATCH; ++x) {
                // the first piece lies in slot 1 of its CTA, the others in slot 0
                const size_t at = ((size_t)(j.cta0 + min(x0 + x, j.pieces - 1)) * 2 + (x0 + x == 0 ? 1 : 0)) * A8_SLOT_HEADS + h;
                ml[x] = __ldcg(reinterpret_cast<const float2*>(p.ws_ml) + at);
                v[x] = __ldcg(reinterpret_cast<const float4*>(p.ws_acc + at * D + e));
            }
#pragma unroll
            for (int x = 0; x < BATCH; ++x) {
                if (x0 + x >= j.pieces) continue;
                const float now = fmaxf(top, ml[x].x), ref = now == -INFINITY ? 0.0f : now;
                const float old = a8_ex2(top - ref), wgt = a8_ex2(ml[x].x - ref);
                sum.x = sum.x * old + v[x].x * wgt; sum.y = sum.y * old + v[x].y * wgt;
                sum.z = sum.z * old + v[x].z * wgt; sum.w = sum.w * old + v[x].w * wgt;
                den = den * old + ml[x].y * wgt;
                top = now;
            }
        }
        a8_write4(p, j.row, ((size_t)j.row * p.nq + j.h0 + h) * D + e, sum, den);
    }
}

template <int D, bool E4M3>
static int a8_launch(const A8Params& p, int ctas, cudaStream_t stream) {
    const size_t smem = sizeof(A8Shared<D>);
    static bool configured[64] = {};                          // per device: the attribute belongs to a device's copy of the kernel
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return pi_refuse("pi_attention_decode_8bit: no current device below 64");
    if (!configured[device]) {
        cudaError_t err = cudaFuncSetAttribute(attn_decode_8bit_kernel<D, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (err != cudaSuccess) {
            snprintf(g_pi_error, sizeof(g_pi_error), "pi_attention_decode_8bit: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(err));
            return (int)err;
        }
        configured[device] = true;
    }
    pi_launch(attn_decode_8bit_kernel<D, E4M3>, dim3((unsigned)ctas), dim3(A8_THREADS), smem, stream, p);
    return pi_check_launch("pi_attention_decode_8bit");
}

// arguments as one record of 8-byte fields
struct A8Args {
    const void* q; long long q_stride; const void* kcache; const void* vcache; const float* kscale; const float* vscale;
    long long cache_dtype, num_pages; const int* block_table; long long bt_rows, bt_stride;
    const int* seg_off; const int* seg_slot; const int* seg_start; const int* seg_len; void* out;
    float* ws_acc; float* ws_ml; void* ws_count; long long ws_ctas, span_min, pair_cost;
    long long num_tokens, num_segments, nq, nkv, head_dim, page_size, window;
    double scale;
};

PI_EXPORT int pi_attention_decode_8bit(const A8Args* args, cudaStream_t stream) {
    const A8Args& a = *args;
    const int q_stride = (int)a.q_stride, cache_dtype = (int)a.cache_dtype, bt_rows = (int)a.bt_rows, bt_stride = (int)a.bt_stride;
    const int ws_ctas = (int)a.ws_ctas, span_min = (int)a.span_min, pair_cost = (int)a.pair_cost, num_tokens = (int)a.num_tokens;
    const int num_segments = (int)a.num_segments, nq = (int)a.nq, nkv = (int)a.nkv, head_dim = (int)a.head_dim;
    const int page_size = (int)a.page_size, window = (int)a.window;
    const float scale = (float)a.scale;
    if (num_segments <= 0 || num_tokens <= 0) return 0;
    if (head_dim != 64 && head_dim != 128) return pi_refuse("pi_attention_decode_8bit: head size %d is not 64 or 128", head_dim);
    if (!(scale > 0.0f)) return pi_refuse("pi_attention_decode_8bit: the score scale must be positive");
    if (nq <= 0 || nkv <= 0 || nq % nkv != 0) return pi_refuse("pi_attention_decode_8bit: nq=%d must be a positive multiple of nkv=%d", nq, nkv);
    if (num_segments > A8_MAX_SEGS) return pi_refuse("pi_attention_decode_8bit: %d segments; this kernel takes at most %d", num_segments, A8_MAX_SEGS);
    if (page_size < C8_BLOCK || (page_size & (page_size - 1))) return pi_refuse("pi_attention_decode_8bit: page size %d must be a power of two of at least 16", page_size);
    if (cache_dtype != PI_E4M3 && cache_dtype != PI_INT8) return pi_refuse("pi_attention_decode_8bit: unknown dtype code %d of the pages", cache_dtype);
    if (window < 0 || bt_rows <= 0 || bt_stride <= 0) return pi_refuse("pi_attention_decode_8bit: window=%d, block table [%d, %d]", window, bt_rows, bt_stride);
    if (ws_ctas <= 0 || ws_ctas > 256 || a.ws_acc == nullptr || a.ws_ml == nullptr || a.ws_count == nullptr) return pi_refuse("pi_attention_decode_8bit: the workspace is missing (or for more than 256 CTAs: %d)", ws_ctas);
    // (span_min and the units, at most 10^9 each, are added up in 32 bits)
    if (a.span_min < 1 || a.span_min > 1000000000LL || a.pair_cost < 0 || a.pair_cost > 64) return pi_refuse("pi_attention_decode_8bit: span_min=%lld must lie between 1 and 10^9 and pair_cost=%lld between 0 and 64", a.span_min, a.pair_cost);
    if (q_stride % 8 != 0 || (((uintptr_t)a.q | (uintptr_t)a.kcache | (uintptr_t)a.vcache) & 15) || ((uintptr_t)a.out & 7))
        return pi_refuse("pi_attention_decode_8bit: q and the pages must start on 16-byte boundaries, the output on an 8-byte one, and q needs a stride that is a multiple of 8");
    const long long blocks = a.num_pages * nkv * (page_size / C8_BLOCK);
    if (a.num_pages <= 0 || blocks > 2147483647LL) return pi_refuse("pi_attention_decode_8bit: %lld pages are %lld blocks: beyond the limit", a.num_pages, blocks);
    if ((long long)bt_stride * page_size > 2147483647LL - 2 * A8_TILE * A8_WARPS * 4)
        return pi_refuse("pi_attention_decode_8bit: block tables of %d pages are beyond the limit", bt_stride);
    A8Params p;
    p.q = (const bf16*)a.q; p.q_stride = q_stride;
    p.kcache = (const unsigned char*)a.kcache; p.vcache = (const unsigned char*)a.vcache; p.kscale = a.kscale; p.vscale = a.vscale;
    p.block_table = a.block_table; p.bt_rows = bt_rows; p.bt_stride = bt_stride;
    p.seg_off = a.seg_off; p.seg_slot = a.seg_slot; p.seg_start = a.seg_start; p.seg_len = a.seg_len;
    p.out = (bf16*)a.out; p.ws_acc = a.ws_acc; p.ws_ml = a.ws_ml; p.ws_count = (unsigned*)a.ws_count;
    p.num_pages = (int)a.num_pages; p.num_tokens = num_tokens; p.num_segments = num_segments;
    p.nq = nq; p.nkv = nkv; p.group = nq / nkv; p.head_tiles = (p.group + A8_HEADS - 1) / A8_HEADS;
    p.window = window; p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.span_min = span_min; p.pair_cost = pair_cost;
    p.scale_log2 = scale * 1.4426950408889634f;
    long long seg_tiles = ((long long)bt_stride * page_size + A8_TILE - 1) / A8_TILE;
    if (window > 0 && seg_tiles > window / A8_TILE + 2) seg_tiles = window / A8_TILE + 2;
    const long long units = (long long)num_segments * nkv * p.head_tiles * (seg_tiles + pair_cost);
    if (units > 1000000000LL) return pi_refuse("pi_attention_decode_8bit: up to %lld tiles of keys are beyond the limit", units);
    if (head_dim == 128) return cache_dtype == PI_E4M3 ? a8_launch<128, true>(p, ws_ctas, stream) : a8_launch<128, false>(p, ws_ctas, stream);
    return cache_dtype == PI_E4M3 ? a8_launch<64, true>(p, ws_ctas, stream) : a8_launch<64, false>(p, ws_ctas, stream);
}
