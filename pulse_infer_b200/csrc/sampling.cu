// Token selection on the device from 32-bit logits: greedy (argmax) and temperature sampling with
// optional top-k and top-p, one thread block per row, plus one kernel that applies all rules of a request to its row
// in one pass (penalties over the token history, biases, banned ids, a mask of allowed ids) and a small one that edits
// single logits in place (an operator of its own; the sampler uses the rules).
//
// Reference parity (the reference samples on the CPU):
//   greedy       src/scheduler/continuous_batch_engine.cpp:20-62   strict '>' so the lowest index wins ties
//   temperature  demo/qwen3_infer.cpp:382-393   weight = exp((logit - max) / temperature); <= 0 means greedy
//   top-k        demo/qwen3_infer.cpp:336-358   the k largest; among equal logits the earlier index stays
//   top-p        demo/qwen3_infer.cpp:395-409   shortest prefix (by descending logit) with cumulative mass >= p
//   draw         demo/qwen3_infer.cpp:411-422   uniform in [0, total), first candidate with cumulative >= draw
//   penalty/ban  demo/qwen3_infer.cpp:251-264, 522-535
// A row in which no token is left - every logit is -inf, by rules, or NaN - gives -1, which ends a request.
// Differences by design: the draw comes from a counter-based generator keyed by (seed, draw index) so a
// request's tokens do not depend on batching; the cumulative walk is in index order rather than sorted
// order (the distribution is the same); all logits equal to the top-p threshold are kept.
#include <limits.h>
#include <math.h>

#include "common.cuh"

__device__ __forceinline__ unsigned ordered_key(float f) {
    // monotone map float -> unsigned (NaN sorts lowest so it is never chosen)
    if (f != f) return 0u;
    const unsigned u = __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

#define KEY_MINUS_INF 0x007fffffu      // ordered_key(-INFINITY)

__device__ __forceinline__ unsigned long long splitmix64(unsigned long long z) {
    z += 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

// uniform in [0, 1) with 24 bits, from (seed, counter)
__device__ __forceinline__ float uniform_from(unsigned long long seed, unsigned long long counter) {
    const unsigned long long r = splitmix64(splitmix64(seed) ^ (counter * 0xD1342543DE82EF95ull));
    return (float)(r >> 40) * (1.0f / 16777216.0f);
}

struct ArgMax { float v; int i; };
__device__ __forceinline__ ArgMax better(ArgMax a, ArgMax b) {
    if (b.i < 0) return a;
    if (a.i < 0) return b;
    if (b.v > a.v || (b.v == a.v && b.i < a.i)) return b;
    return a;
}

// index -1 where there is nothing to choose: a logit of -inf is a forbidden token, NaN is none
__device__ ArgMax block_argmax(const float* __restrict__ x, int n, ArgMax* sh /* 33 */) {
    ArgMax best = {-INFINITY, -1};
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const float v = x[i];
        if (v > best.v) { best.v = v; best.i = i; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        ArgMax other;
        other.v = __shfl_xor_sync(0xffffffffu, best.v, o);
        other.i = __shfl_xor_sync(0xffffffffu, best.i, o);
        best = better(best, other);
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = (blockDim.x + 31) >> 5;
    if (lane == 0) sh[warp] = best;
    __syncthreads();
    if (warp == 0) {
        ArgMax t = lane < nwarps ? sh[lane] : ArgMax{-INFINITY, -1};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            ArgMax other;
            other.v = __shfl_xor_sync(0xffffffffu, t.v, o);
            other.i = __shfl_xor_sync(0xffffffffu, t.i, o);
            t = better(t, other);
        }
        if (lane == 0) sh[32] = t;
    }
    __syncthreads();
    const ArgMax r = sh[32];
    __syncthreads();
    return r;
}

__global__ void argmax_kernel(const float* __restrict__ logits, int ld, int vocab, int* __restrict__ out) {
    __shared__ ArgMax sh[33];
    pdl_wait();
    pdl_trigger();
    const ArgMax r = block_argmax(logits + (size_t)blockIdx.x * ld, vocab, sh);
    if (threadIdx.x == 0) out[blockIdx.x] = r.i;
}

// Large vocabularies: a row is cut into slices scanned by separate blocks (one block per row would leave
// most of the GPU idle and take tens of microseconds), then one small block per row picks among the slices.
#define ARGMAX_SLICE 4096
__global__ void argmax_slices_kernel(const float* __restrict__ logits, int ld, int vocab, float* __restrict__ cand_val,
                                     int* __restrict__ cand_idx, int slices) {
    __shared__ ArgMax sh[33];
    pdl_wait();
    pdl_trigger();
    const int row = blockIdx.y, slice = blockIdx.x;
    const int begin = slice * ARGMAX_SLICE;
    const int n = min(ARGMAX_SLICE, vocab - begin);
    ArgMax r = block_argmax(logits + (size_t)row * ld + begin, n, sh);
    if (threadIdx.x == 0) {
        cand_val[row * slices + slice] = r.v;
        cand_idx[row * slices + slice] = r.i < 0 ? -1 : r.i + begin;
    }
}

__global__ void argmax_pick_kernel(const float* __restrict__ cand_val, const int* __restrict__ cand_idx, int slices,
                                   int* __restrict__ out) {
    pdl_wait();
    pdl_trigger();
    const int row = blockIdx.x;
    ArgMax best = {-INFINITY, -1};
    for (int i = threadIdx.x; i < slices; i += 32) {   // ascending index per lane; ties keep the lower index
        ArgMax c = {cand_val[row * slices + i], cand_idx[row * slices + i]};
        best = better(best, c);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        ArgMax other;
        other.v = __shfl_xor_sync(0xffffffffu, best.v, o);
        other.i = __shfl_xor_sync(0xffffffffu, best.i, o);
        best = better(best, other);
    }
    if (threadIdx.x == 0) out[row] = best.i;
}

PI_EXPORT int pi_argmax_scratch_floats(int rows, int vocab) {
    const int slices = (vocab + ARGMAX_SLICE - 1) / ARGMAX_SLICE;
    return vocab >= 4 * ARGMAX_SLICE ? 2 * rows * slices : 0;
}

// scratch: pi_argmax_scratch_floats(rows, vocab) 4-byte words (may be null when that is 0)
PI_EXPORT int pi_argmax(const float* logits, int ld, int rows, int vocab, int* out, void* scratch, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (vocab <= 0 || ld < vocab) return pi_refuse("pi_argmax: vocab=%d ld=%d", vocab, ld);
    if (vocab >= 4 * ARGMAX_SLICE) {
        if (scratch == nullptr) return pi_refuse("pi_argmax: scratch is missing");
        if (rows > 65535) return pi_refuse("pi_argmax: %d rows are beyond the grid limit", rows);
        const int slices = (vocab + ARGMAX_SLICE - 1) / ARGMAX_SLICE;
        float* cand_val = (float*)scratch;
        int* cand_idx = (int*)scratch + (size_t)rows * slices;
        pi_launch(argmax_slices_kernel, dim3(slices, rows), dim3(256), 0, stream, logits, ld, vocab, cand_val, cand_idx, slices);
        pi_launch(argmax_pick_kernel, dim3(rows), dim3(32), 0, stream, (const float*)cand_val, (const int*)cand_idx, slices, out);
    } else {
        pi_launch(argmax_kernel, dim3(rows), dim3(vocab >= 4096 ? 1024 : 256), 0, stream, logits, ld, vocab, out);
    }
    return pi_check_launch("pi_argmax");
}

// exclusive scan over the block in thread order; returns the exclusive prefix, *total gets the sum
template <typename T>
__device__ T block_exclusive_scan(T v, T* sh /* 33 */, T* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = (blockDim.x + 31) >> 5;
    T incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T n = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += n;
    }
    if (lane == 31) sh[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        T w = lane < nwarps ? sh[lane] : (T)0;
        T wi = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const T n = __shfl_up_sync(0xffffffffu, wi, o);
            if (lane >= o) wi += n;
        }
        sh[lane] = wi - w;  // exclusive prefix of the warps
        if (lane == 31) sh[32] = wi;
    }
    __syncthreads();
    const T result = sh[warp] + (incl - v);
    *total = sh[32];
    __syncthreads();
    return result;
}

__global__ void sample_kernel(const float* __restrict__ logits, int ld, int vocab, const float* __restrict__ temperature,
                              const int* __restrict__ top_k, const float* __restrict__ top_p,
                              const unsigned long long* __restrict__ seeds,
                              const unsigned long long* __restrict__ counters, int* __restrict__ out,
                              const long long* __restrict__ row_entry) {
    __shared__ ArgMax sh_arg[33];
    __shared__ float sh_f[33];
    __shared__ int sh_i[33];
    __shared__ int sh_pick;
    pdl_wait();
    pdl_trigger();
    const int row = blockIdx.x;
    const float* x = logits + (size_t)row * ld;
    const ArgMax top = block_argmax(x, vocab, sh_arg);
    // Without row_entry the options of row r sit at index r.  With it, row_entry[2r] names the entry of the option
    // tables that row r uses (tables filled once per set of options) and row_entry[2r + 1] is its draw counter.
    const int entry = row_entry != nullptr ? (int)row_entry[2 * row] : row;
    const unsigned long long counter = row_entry != nullptr ? (unsigned long long)row_entry[2 * row + 1] : counters[row];
    const float temp = temperature[entry];
    if (temp <= 0.0f || top.i < 0 || top.v == INFINITY) {      // +inf has all of the probability
        if (threadIdx.x == 0) out[row] = top.i;
        return;
    }
    const int chunk = (vocab + blockDim.x - 1) / blockDim.x;
    const int c0 = threadIdx.x * chunk, c1 = min(vocab, c0 + chunk);

    // ---- top-k: the key of the k-th largest logit, and up to which index equal logits are kept ----------
    const int k = top_k[entry];
    unsigned key_k = 0u;       // keep keys > key_k, and keys == key_k with index <= tie_cut
    int tie_cut = INT_MAX;
    if (k > 0 && k < vocab) {
        for (int bit = 31; bit >= 0; --bit) {
            const unsigned cand = key_k | (1u << bit);
            float cnt = 0.0f;
            for (int i = threadIdx.x; i < vocab; i += blockDim.x) cnt += ordered_key(x[i]) >= cand ? 1.0f : 0.0f;
            cnt = block_sum(cnt, sh_f);  // counts up to 2^24 are exact in float
            if (cnt >= (float)k) key_k = cand;
        }
        float gt = 0.0f;
        for (int i = threadIdx.x; i < vocab; i += blockDim.x) gt += ordered_key(x[i]) > key_k ? 1.0f : 0.0f;
        const int ties_allowed = k - (int)block_sum(gt, sh_f);
        int mine = 0;
        for (int i = c0; i < c1; ++i) mine += ordered_key(x[i]) == key_k;
        int total_ties;
        const int before = block_exclusive_scan<int>(mine, sh_i, &total_ties);
        if (threadIdx.x == 0) sh_pick = INT_MAX;
        __syncthreads();
        if (ties_allowed < total_ties && before < ties_allowed && before + mine >= ties_allowed) {
            int seen = before;
            for (int i = c0; i < c1; ++i)
                if (ordered_key(x[i]) == key_k && ++seen == ties_allowed) { sh_pick = i; break; }
        }
        __syncthreads();
        tie_cut = sh_pick;
        __syncthreads();
    }
    // NaN and -inf (a forbidden token) are never kept: a weight of zero could be drawn, by a draw of exactly zero or where the
    // sums round; with no top-k, key_k stays 0 and every other number is kept
    auto kept_k = [&](int i, unsigned key) { return key > KEY_MINUS_INF && (key > key_k || (key == key_k && i <= tie_cut)); };
    const float inv_t = 1.0f / temp;

    // ---- top-p: the largest value v whose upper mass (logit >= v, inside the top-k set) reaches p * Z ---
    const float pp = top_p[entry];
    unsigned key_p = 0u;
    if (pp > 0.0f && pp < 1.0f) {
        float z = 0.0f;
        for (int i = threadIdx.x; i < vocab; i += blockDim.x)
            if (kept_k(i, ordered_key(x[i]))) z += expf((x[i] - top.v) * inv_t);
        z = block_sum(z, sh_f);
        const float want = pp * z;
        for (int bit = 31; bit >= 0; --bit) {
            const unsigned cand = key_p | (1u << bit);
            float mass = 0.0f;
            for (int i = threadIdx.x; i < vocab; i += blockDim.x) {
                const unsigned key = ordered_key(x[i]);
                if (key >= cand && kept_k(i, key)) mass += expf((x[i] - top.v) * inv_t);
            }
            mass = block_sum(mass, sh_f);
            if (mass >= want) key_p = cand;
        }
    }

    // ---- draw: first index (in index order) whose cumulative kept weight reaches u * total --------------
    float mine = 0.0f;
    int last_kept = -1;
    for (int i = c0; i < c1; ++i) {
        const unsigned key = ordered_key(x[i]);
        if (key >= key_p && kept_k(i, key)) { mine += expf((x[i] - top.v) * inv_t); last_kept = i; }
    }
    float total;
    const float before = block_exclusive_scan<float>(mine, sh_f, &total);
    const float target = uniform_from(seeds[entry], counter) * total;
    if (threadIdx.x == 0) sh_pick = INT_MAX;
    __syncthreads();
    int pick = INT_MAX;
    if (last_kept >= 0 && before + mine >= target) {
        float run = before;
        pick = last_kept;
        for (int i = c0; i < c1; ++i) {
            const unsigned key = ordered_key(x[i]);
            if (key >= key_p && kept_k(i, key)) {
                run += expf((x[i] - top.v) * inv_t);
                if (run >= target) { pick = i; break; }
            }
        }
    }
    if (pick != INT_MAX) atomicMin(&sh_pick, pick);
    __syncthreads();
    int result = sh_pick;
    __syncthreads();
    if (result == INT_MAX) {  // rounding left the target beyond every prefix: take the last kept index
        if (threadIdx.x == 0) sh_pick = -1;
        __syncthreads();
        if (last_kept >= 0) atomicMax(&sh_pick, last_kept);
        __syncthreads();
        result = sh_pick;
    }
    if (threadIdx.x == 0) out[row] = result;
}

PI_EXPORT int pi_sample(const float* logits, int ld, int rows, int vocab, const float* temperature, const int* top_k,
                        const float* top_p, const unsigned long long* seeds, const unsigned long long* counters,
                        int* out, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (vocab <= 0 || ld < vocab) return pi_refuse("pi_sample: vocab=%d ld=%d", vocab, ld);
    if (vocab > (1 << 24)) return pi_refuse("pi_sample: vocab=%d is beyond 2^24", vocab);
    pi_launch(sample_kernel, dim3(rows), dim3(vocab >= 4096 ? 1024 : 256), 0, stream, logits, ld, vocab, temperature, top_k,
              top_p, seeds, counters, out, (const long long*)nullptr);
    return pi_check_launch("pi_sample");
}

// The same with the options in tables of `entries` entries that outlive the step: row r uses entry row_entry[2r]
// and draw counter row_entry[2r + 1] (int64 pairs: the only per-step data, one small copy).
PI_EXPORT int pi_sample_entries(const float* logits, int ld, int rows, int vocab, const float* temperature, const int* top_k,
                                const float* top_p, const unsigned long long* seeds, const long long* row_entry,
                                int* out, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (vocab <= 0 || ld < vocab) return pi_refuse("pi_sample_entries: vocab=%d ld=%d", vocab, ld);
    if (vocab > (1 << 24)) return pi_refuse("pi_sample_entries: vocab=%d is beyond 2^24", vocab);
    if (row_entry == nullptr) return pi_refuse("pi_sample_entries: the (entry, counter) pairs are missing");
    pi_launch(sample_kernel, dim3(rows), dim3(vocab >= 4096 ? 1024 : 256), 0, stream, logits, ld, vocab, temperature, top_k,
              top_p, seeds, (const unsigned long long*)nullptr, out, row_entry);
    return pi_check_launch("pi_sample_entries");
}

// logits[rows[i], tokens[i]] = set ? values[i] : logits[...] + values[i]; (row, token) pairs must be distinct
__global__ void logit_edit_kernel(float* __restrict__ logits, int ld, int vocab, const int* __restrict__ rows,
                                  const int* __restrict__ tokens, const float* __restrict__ values, int n, int set) {
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int tok = tokens[i];
    if (tok < 0 || tok >= vocab) return;
    float* dst = logits + (size_t)rows[i] * ld + tok;
    *dst = set ? values[i] : *dst + values[i];
}

PI_EXPORT int pi_logit_edit(float* logits, int ld, int vocab, const int* rows, const int* tokens, const float* values,
                            int n, int set, cudaStream_t stream) {
    if (n <= 0) return 0;
    pi_launch(logit_edit_kernel, dim3((n + 127) / 128), dim3(128), 0, stream, logits, ld, vocab, rows, tokens, values, n, set);
    return pi_check_launch("pi_logit_edit");
}

// ---------------------------------------------------------------------------------------------------
// The rules of each row on its logits, in one pass.  With the row's history h (its first prompt_len entries the prompt),
// seen = v occurs in h, count = occurrences behind the prompt, for every token id v
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * count - (seen ? presence : 0) + bias[v],   x = -inf where the row's mask has a zero bit
// A bias of -inf forbids the id, whatever its logit is.  Of several biases of a row for one id the last counts; ids outside the vocabulary are passed over.
//
// The logits are read and written once (4 + 4 bytes each: what bounds a large step); a step of one row is bound by latency.
// A block owns RULE_SLICE ids of a row.  It asks for their logits; while they come it counts the history's ids of its slice in
// shared memory (every block of the row walks the whole history out of L2; integer atomics, so the order does not matter), and
// applies the rules as it stores.  No workspace, no second launch.
// Measured (B200, 152k logits): 3.3 us for a row with a history of 4,000; 23 us for 64 rows with histories to 8,000, 300 biases
// and masks (12.2 us of traffic; 11.5 us without any rule, so the walks and marks are the rest).  Slices of 4,096 ids for 256
// threads: 3.5 and 24.4 us (more walks); 8,192 for 512, with 64 KB of shared memory: 3.5 and 22.3 us; 12,288 for 768: 4.1 and
// 23.9; the first history entries asked for before the logits: 23.9.  Tried and slower: the
// history walked once by a cluster of eight blocks that mark through distributed shared memory (32 us); a copy kernel and a
// second one with a block per 49,152 ids that changes only the marked ids (28 us); several slices one after the other in a
// block (48 us); divisions by the penalty instead of products with its reciprocal (29 us: nearly every warp has a marked id).
// ---------------------------------------------------------------------------------------------------
#define RULE_THREADS 384
#define RULE_SLICE 6144
#define RULE_VECS (RULE_SLICE / 4 / RULE_THREADS)
#define RULE_BATCH 8            // history entries a thread has in flight

struct RuleParams {
    const float* logits; long long ld; float* out; long long out_ld; int vocab, vec;
    const int* history; const int* history_off; int history_total; const int* prompt_len;
    const float* repetition; const float* frequency; const float* presence;
    const int* bias_off; const int* bias_tokens; const float* bias_values; int bias_total;
    const unsigned* mask; int mask_rows, mask_words; const int* mask_row;
};

// visits every history entry of [from, to) that lies in the slice, RULE_BATCH entries per thread and round trip
template <typename Visit>
__device__ __forceinline__ void rule_walk(const int* history, int from, int to, int begin, int n, Visit&& visit) {
    for (int first = from + threadIdx.x; first < to; first += RULE_BATCH * RULE_THREADS) {
        int tok[RULE_BATCH];
#pragma unroll
        for (int k = 0; k < RULE_BATCH; ++k) tok[k] = first + k * RULE_THREADS < to ? history[first + k * RULE_THREADS] : -1;
#pragma unroll
        for (int k = 0; k < RULE_BATCH; ++k) {
            const unsigned at = (unsigned)tok[k] - (unsigned)begin;
            if (at < (unsigned)n) visit(at);
        }
    }
}

template <bool BIAS>
__global__ void __launch_bounds__(RULE_THREADS, 4) logit_rules_kernel(const RuleParams p) {
    __shared__ __align__(16) unsigned mark[RULE_SLICE];        // bit 31: in the prompt, bit 30: has a bias; below: count behind it
    __shared__ __align__(16) int bias_at[BIAS ? RULE_SLICE : 4];   // index + 1 of the last bias for the id
    pdl_wait();
    pdl_trigger();
    const int row = blockIdx.y, begin = blockIdx.x * RULE_SLICE, n = min(RULE_SLICE, p.vocab - begin);
    const int h0 = max(0, min(p.history_off[row], p.history_total)), h1 = max(h0, min(p.history_off[row + 1], p.history_total));
    const int gen = max(h0, (int)min((long long)h1, (long long)h0 + p.prompt_len[row]));
    int b0 = 0, b1 = 0;
    if (BIAS) { b0 = max(0, min(p.bias_off[row], p.bias_total)); b1 = max(b0, min(p.bias_off[row + 1], p.bias_total)); }
    const float rep = p.repetition[row], freq = p.frequency[row], pres = p.presence[row];
    const int mrow = p.mask != nullptr ? p.mask_row[row] : -1;
    const unsigned* words = mrow >= 0 && mrow < p.mask_rows ? p.mask + (size_t)mrow * p.mask_words + begin / 32 : nullptr;
    const float* x = p.logits + (size_t)row * p.ld + begin;
    float* y = p.out + (size_t)row * p.out_ld + begin;
    int bias_id = BIAS && b0 + (int)threadIdx.x < b1 ? p.bias_tokens[b0 + threadIdx.x] : -1;
    float4 v[RULE_VECS];
#pragma unroll
    for (int k = 0; k < RULE_VECS; ++k) {
        const int i = 4 * (k * RULE_THREADS + threadIdx.x);
        if (p.vec && i + 4 <= n) {
            v[k] = *reinterpret_cast<const float4*>(x + i);
        } else {
            v[k].x = i < n ? x[i] : 0.0f; v[k].y = i + 1 < n ? x[i + 1] : 0.0f;
            v[k].z = i + 2 < n ? x[i + 2] : 0.0f; v[k].w = i + 3 < n ? x[i + 3] : 0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < RULE_VECS; ++k) {
        const int i = k * RULE_THREADS + threadIdx.x;
        reinterpret_cast<uint4*>(mark)[i] = make_uint4(0u, 0u, 0u, 0u);
        if (BIAS) reinterpret_cast<int4*>(bias_at)[i] = make_int4(0, 0, 0, 0);
    }
    __syncthreads();
    if (BIAS) {
        for (int b = b0 + threadIdx.x; b < b1; b += RULE_THREADS) {
            const unsigned at = (unsigned)bias_id - (unsigned)begin;
            if (at < (unsigned)n) { atomicMax(&bias_at[at], b + 1); atomicOr(&mark[at], 0x40000000u); }
            bias_id = b + RULE_THREADS < b1 ? p.bias_tokens[b + RULE_THREADS] : -1;
        }
    }
    rule_walk(p.history, h0, gen, begin, n, [&](unsigned at) { atomicOr(&mark[at], 0x80000000u); });
    rule_walk(p.history, gen, h1, begin, n, [&](unsigned at) { atomicAdd(&mark[at], 1u); });
    __syncthreads();
    const float inv_rep = 1.0f / rep;
#pragma unroll
    for (int k = 0; k < RULE_VECS; ++k) {
        const int i = 4 * (k * RULE_THREADS + threadIdx.x);
        if (i >= n) continue;
        const unsigned bits = words != nullptr ? words[i >> 5] >> (i & 31) : 0xfu;
        const uint4 marks = reinterpret_cast<const uint4*>(mark)[i >> 2];
        float e[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
        if ((marks.x | marks.y | marks.z | marks.w) != 0u) {           // some of the four have a rule of their own
            const unsigned mk[4] = {marks.x, marks.y, marks.z, marks.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float changed = e[c] * (e[c] > 0.0f ? inv_rep : rep) - freq * (float)(mk[c] & 0x3fffffffu) - pres;
                e[c] = (mk[c] & 0xbfffffffu) != 0u ? changed : e[c];
                if (BIAS && (mk[c] & 0x40000000u)) {
                    const float bias = p.bias_values[bias_at[i + c] - 1];
                    e[c] = bias == -INFINITY ? bias : e[c] + bias;          // forbidden, whatever the logit is
                }
            }
        }
        const float4 o = make_float4(bits & 1u ? e[0] : -INFINITY, bits & 2u ? e[1] : -INFINITY, bits & 4u ? e[2] : -INFINITY,
                                     bits & 8u ? e[3] : -INFINITY);
        if (p.vec && i + 4 <= n) {
            *reinterpret_cast<float4*>(y + i) = o;
        } else {
            y[i] = o.x;
            if (i + 1 < n) y[i + 1] = o.y;
            if (i + 2 < n) y[i + 2] = o.z;
            if (i + 3 < n) y[i + 3] = o.w;
        }
    }
}

// arguments as one record of 8-byte fields
struct RuleArgs {
    const float* logits; long long ld; float* out; long long out_ld, rows, vocab;
    const int* history; const int* history_off; long long history_total; const int* prompt_len;
    const float* repetition; const float* frequency; const float* presence;
    const int* bias_off; const int* bias_tokens; const float* bias_values; long long bias_total;
    const void* mask; long long mask_rows; const int* mask_row;
};

PI_EXPORT int pi_logit_rules(const RuleArgs* args, cudaStream_t stream) {
    const RuleArgs& a = *args;
    const float* logits = a.logits;
    float* out = a.out;
    const long long ld = a.ld, out_ld = a.out_ld, history_total = a.history_total, bias_total = a.bias_total;
    const int rows = (int)a.rows, vocab = (int)a.vocab;
    if (rows <= 0) return 0;
    if (vocab <= 0 || ld < vocab || out_ld < vocab) return pi_refuse("pi_logit_rules: vocab=%d ld=%lld out_ld=%lld", vocab, ld, out_ld);
    if (rows > 65535) return pi_refuse("pi_logit_rules: %d rows are beyond the grid limit", rows);
    if (vocab > 2147483647 - RULE_SLICE) return pi_refuse("pi_logit_rules: vocab=%d is beyond the limit", vocab);
    // a count of an id stays below bit 30 of its mark
    if (history_total >= (1 << 30) || bias_total > (1 << 30)) return pi_refuse("pi_logit_rules: histories of %lld or %lld biases are beyond the limit", history_total, bias_total);
    RuleParams p;
    p.logits = logits; p.ld = ld; p.out = out; p.out_ld = out_ld; p.vocab = vocab;
    p.vec = (ld % 4 == 0 && out_ld % 4 == 0 && (((uintptr_t)logits | (uintptr_t)out) & 15) == 0) ? 1 : 0;
    p.history = a.history; p.history_off = a.history_off; p.history_total = (int)history_total; p.prompt_len = a.prompt_len;
    p.repetition = a.repetition; p.frequency = a.frequency; p.presence = a.presence;
    p.bias_off = a.bias_off; p.bias_tokens = a.bias_tokens; p.bias_values = a.bias_values; p.bias_total = (int)bias_total;
    p.mask = (const unsigned*)a.mask; p.mask_rows = (int)a.mask_rows; p.mask_words = (vocab + 31) / 32; p.mask_row = a.mask_row;
    const dim3 grid((vocab + RULE_SLICE - 1) / RULE_SLICE, rows), threads(RULE_THREADS);
    if (a.bias_off != nullptr) pi_launch(logit_rules_kernel<true>, grid, threads, 0, stream, p);
    else pi_launch(logit_rules_kernel<false>, grid, threads, 0, stream, p);
    return pi_check_launch("pi_logit_rules");
}
