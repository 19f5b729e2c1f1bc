// Log probabilities of given tokens, the entropy of each row and the most likely tokens with theirs, from logits that are read
// once.
//
//   lse = m + ln s,  s = sum e^(x - m);   logprob(j) = x_j - lse;   entropy = ln s - t / s,  t = sum e^(x - m) (x - m)
//
// (t / s is the mean of x - m under the distribution: neither term carries the size of the logits.)  A thread keeps m, s and t of
// its own elements, worked out in base 2 over 32 of them at a time, so that most passes rescale nothing; threads, warps and the
// blocks of a cluster join theirs in a fixed order.
//
// The k most likely tokens need no second pass over the row.  A thread's maximum is m, which it has anyway, and where it stands
// is looked up only when it moves.  The k-th largest of the maxima of the 64 groups of four threads is a bound with at least k
// elements at or above it, and only batches of 32 whose maximum (kept in shared memory) is at or above it can hold one: about
// k of a row's 2,048, which are read again.  (Without the batches' maxima a thread's whole 256 elements are, 32-byte sectors for
// 16-byte pieces: 2,047 rows of 65,536 with 20 alternatives 117 us, 82 without alternatives.)  What they find is ranked by comparison, by (logit descending, id ascending) in
// one 64-bit key, so that the result does not depend on the order in which it was found.  If more is found than the list holds
// (rows made for it), the k largest are taken one after the other.
//
// Few rows: up to 8 blocks share a row as a cluster and join through its shared memory (8 rows of 65,536: 10.4 us on one block
// each, 7.5 on eight, 9.1 on sixteen); from one block a multiprocessor on a block has its row for itself (300 rows: 22 us, on two
// 22, on four 29).
#include "common.cuh"
#include "cluster.cuh"

using namespace vapi;

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_GROUPS = LP_THREADS / 4;
constexpr int LP_MAX_TOP = 64;                     // alternatives at most (as many as there are groups)
constexpr int LP_LIST = 1024;
constexpr int LP_SLOTS = 16;                       // batches whose maxima are kept apart (the 17th shares with the first, and so on)
constexpr int LP_MAX_CLUSTER = 8;
// a distance in powers of two at which nothing is left of a term (2^-126 is the smallest that ex2 gives), kept finite so that zero times it is zero
constexpr float LP_FAR = -200.f;
constexpr float LN2 = 0.6931471805599453f, LOG2E = 1.4426950408889634f;

typedef unsigned long long Key;
// larger logits first, then smaller ids; 0: nothing (a NaN is never an alternative)
__device__ __forceinline__ Key lp_key(float x, int id) {
    const unsigned u = __float_as_uint(x + 0.f);   // (the two zeros are one number)
    const unsigned o = x != x ? 0u : ((u & 0x80000000u) ? ~u : u | 0x80000000u);
    return o == 0u ? 0ull : ((Key)o << 32) | (unsigned)~id;
}
__device__ __forceinline__ float lp_logit(Key k) {
    const unsigned o = (unsigned)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int lp_id(Key k) { return (int)~(unsigned)k; }

__device__ __forceinline__ float lp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// a thread's, a warp's or a block's share of the sums, in base 2: m the largest logit, s = sum 2^((x - m) log2 e), t = sum of
// those times (x - m) log2 e
struct Share { float m, s, t; };
__device__ __forceinline__ Share lp_join(const Share& a, const Share& b) {
    Share r;
    r.m = fmaxf(a.m, b.m);
    const float mu = r.m == -INFINITY ? 0.f : r.m;
    const float da = a.m == -INFINITY ? 0.f : fmaxf((a.m - mu) * LOG2E, LP_FAR), db = b.m == -INFINITY ? 0.f : fmaxf((b.m - mu) * LOG2E, LP_FAR);
    const float fa = lp_ex2(da), fb = lp_ex2(db);
    r.s = a.s * fa + b.s * fb;
    r.t = fmaf(a.s, da, a.t) * fa + fmaf(b.s, db, b.t) * fb;
    return r;
}

// the shares of a warp's lanes, joined: onto the largest m first, so that the sums are only added
__device__ __forceinline__ Share lp_warp(const Share& a) {
    Share r;
    r.m = warp_max(a.m);
    const float d = a.m == -INFINITY ? 0.f : fmaxf((a.m - r.m) * LOG2E, LP_FAR), f = lp_ex2(d);
    r.s = warp_sum(a.s * f);
    r.t = warp_sum(fmaf(a.s, d, a.t) * f);
    return r;
}

template <bool V> struct Truth { static constexpr bool value = V; };

template <typename T> struct LpVec;
template <> struct LpVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(p));
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    }
};
template <> struct LpVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[8]) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, 4)
logprobs_kernel(const T* __restrict__ logits, int vocab, long long stride, const int* __restrict__ tokens, int top, float* __restrict__ logprob,
                float* __restrict__ entropy, int* __restrict__ top_ids, float* __restrict__ top_lp, int slices, int* __restrict__ status) {
    constexpr int N = LpVec<T>::N, BATCH = 32 / N;
    __shared__ Share warp_share[LP_WARPS];
    __shared__ Share own_share;                    // this block's, read by the first block of its cluster
    __shared__ Key groups[LP_GROUPS];
    __shared__ Key bound;
    __shared__ Key list[LP_LIST];
    __shared__ Key best[LP_MAX_TOP];               // this block's k largest, in order, read by the first block of its cluster
    __shared__ Key warp_best[LP_WARPS];
    __shared__ float batch_max[LP_SLOTS][LP_THREADS];
    __shared__ unsigned short again[LP_SLOTS * LP_THREADS];       // batches that are looked at again: thread | slot << 8
    __shared__ int n_again, n_list;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = (int)blockIdx.x / slices, slice = (int)blockIdx.x % slices;
    pdl_trigger();
    if (tid == 0) n_again = n_list = 0;
    pdl_wait();
    const T* x = logits + (size_t)row * stride;
    // a row: `head` elements up to the first 16-byte boundary, pieces of 16 bytes, `tail` elements; the pieces are cut into slices
    const int head = min(vocab, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
    const int pieces = (vocab - head) / N, tail = vocab - head - pieces * N;
    const int from = (int)((long long)pieces * slice / slices), upto = (int)((long long)pieces * (slice + 1) / slices);
    const bool has_head = slice == 0 && tid < head, has_tail = slice == slices - 1 && tid < tail;
    const T* body = x + head;

    // ---- one pass: m, s, t of this thread's elements, and where m stands
    Share a = {-INFINITY, 0.f, 0.f};
    int at = has_head ? tid : (from + tid < upto ? head + (from + tid) * N : head + pieces * N + tid);
    auto add = [&](float v, float mu) {            // mu: m, or 0 where nothing but -inf has been seen
        const float d = (v - mu) * LOG2E, e = lp_ex2(d);
        a.s += e;
        a.t = fmaf(e, fmaxf(d, LP_FAR), a.t);      // (an e of zero stays zero beside a logit of -inf)
    };
    auto ground = [&]() { return a.m == -INFINITY ? 0.f : a.m; };
    auto raise = [&](float mx) {                   // a new largest logit: what was summed moves onto it
        const float d = a.m == -INFINITY ? 0.f : fmaxf((a.m - mx) * LOG2E, LP_FAR), f = lp_ex2(d);
        a.t = fmaf(a.s, d, a.t) * f;
        a.s *= f;
        a.m = mx;
    };
    if (has_head) {
        const float v = to_f32(x[tid]);
        if (v > a.m) a.m = v;
        add(v, ground());
    }
    int i = from + tid, slot = 0;
    const int slots = top > 0 ? min(LP_SLOTS, (upto - from + BATCH * LP_THREADS - 1) / (BATCH * LP_THREADS)) : 0;
    for (int k = 0; k < slots; ++k) batch_max[k][tid] = -INFINITY;
    auto batch = [&](auto whole) {                 // 32 elements; not whole: pieces behind the slice are -inf
        float v[BATCH][N];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            if (decltype(whole)::value || i + b * LP_THREADS < upto) {
                LpVec<T>::load(body + (size_t)(i + b * LP_THREADS) * N, v[b]);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) v[b][e] = -INFINITY;
            }
        }
        float mx = v[0][0];
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
#pragma unroll
            for (int e = 0; e < N; ++e) mx = fmaxf(mx, v[b][e]);
        if (top > 0) {
            batch_max[slot][tid] = fmaxf(batch_max[slot][tid], mx);
            slot = slot + 1 < LP_SLOTS ? slot + 1 : 0;
        }
        if (mx > a.m) {
            raise(mx);
            int first = 0;
#pragma unroll
            for (int b = BATCH - 1; b >= 0; --b)
#pragma unroll
                for (int e = N - 1; e >= 0; --e) first = v[b][e] == mx ? b * LP_THREADS * N + e : first;
            at = head + i * N + first;
        }
        const float mu = ground();
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
#pragma unroll
            for (int e = 0; e < N; ++e) add(v[b][e], mu);
        i += BATCH * LP_THREADS;
    };
    while (i + (BATCH - 1) * LP_THREADS < upto) batch(Truth<true>());
    if (i < upto) batch(Truth<false>());
    if (has_tail) {
        const int id = head + pieces * N + tid;
        const float v = to_f32(x[id]);
        if (v > a.m) { raise(v); at = id; }
        add(v, ground());
    }
    const bool any = has_head || from + tid < upto || has_tail;

    // ---- the block's share
    const Share w = lp_warp(a);
    if (lane == 0) warp_share[warp] = w;

    // ---- the block's k largest
    const Key mine = any ? lp_key(a.m, at) : 0ull;
    if (top > 0) {
        Key g = mine;
        Key o = __shfl_xor_sync(0xffffffffu, g, 1);
        g = o > g ? o : g;
        o = __shfl_xor_sync(0xffffffffu, g, 2);
        g = o > g ? o : g;
        if ((lane & 3) == 0) groups[tid >> 2] = g;
        if (tid == 0) bound = 0ull;                // (fewer than k groups with an element: every element is looked at)
    }
    __syncthreads();
    if (warp == LP_WARPS - 1) {
        const Share b = lp_warp(lane < LP_WARPS ? warp_share[lane] : Share{-INFINITY, 0.f, 0.f});
        if (lane == 0) own_share = b;
    }
    if (top > 0) {
        if (tid < LP_GROUPS) {
            const Key g = groups[tid];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < LP_GROUPS; ++j) rank += groups[j] > g;
            if (g != 0ull && rank == top - 1) bound = g;
        }
        __syncthreads();
        const Key least = bound;
        // batches that can hold an element at or above the bound: a larger maximum, or an equal one whose first place is not behind it
        const float least_x = lp_logit(least);
        const int least_id = least == 0ull ? 0x7fffffff : lp_id(least);
        for (int k = 0; k < slots; ++k) {
            const int piece = from + tid + k * BATCH * LP_THREADS;
            const float mx = batch_max[k][tid];
            if (piece < upto && (least == 0ull || mx > least_x || (mx == least_x && head + piece * N <= least_id)))
                again[atomicAdd(&n_again, 1)] = (unsigned short)(tid | k << 8);
        }
        auto offer = [&](Key k) {
            if (k != 0ull && k >= least) {
                const int place = atomicAdd(&n_list, 1);
                if (place < LP_LIST) list[place] = k;
            }
        };
        if (has_head) offer(lp_key(to_f32(x[tid]), tid));
        if (has_tail) offer(lp_key(to_f32(x[head + pieces * N + tid]), head + pieces * N + tid));
        __syncthreads();
        const int n = n_again;
        // the elements of those batches, a batch by 32 / N lanes (one piece each)
        auto visit_all = [&](auto&& visit) {
            for (int j = warp * N + lane / BATCH; j < n; j += LP_WARPS * N) {
                const int t = again[j] & 0xff;
                for (int p = from + t + ((again[j] >> 8) * BATCH + lane % BATCH) * LP_THREADS; p < upto; p += LP_SLOTS * BATCH * LP_THREADS) {
                    float v[N];
                    LpVec<T>::load(body + (size_t)p * N, v);
#pragma unroll
                    for (int e = 0; e < N; ++e) visit(lp_key(v[e], head + p * N + e));
                }
            }
        };
        visit_all(offer);
        if (tid < top) best[tid] = 0ull;
        __syncthreads();
        const int found = n_list;
        if (found <= LP_LIST) {
            for (int j = tid; j < found; j += LP_THREADS) {
                const Key k = list[j];
                int rank = 0;
                for (int c = 0; c < found; ++c) rank += list[c] > k;
                if (rank < top) best[rank] = k;
            }
        } else {
            Key last = ~0ull;
            for (int r = 0; r < top && last != 0ull; ++r) {                 // (the same for all threads)
                Key b = 0ull;
                auto look = [&](Key k) { if (k < last && k > b) b = k; };
                visit_all(look);
                if (has_head) look(lp_key(to_f32(x[tid]), tid));
                if (has_tail) look(lp_key(to_f32(x[head + pieces * N + tid]), head + pieces * N + tid));
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const Key other = __shfl_xor_sync(0xffffffffu, b, o);
                    b = other > b ? other : b;
                }
                if (lane == 0) warp_best[warp] = b;
                __syncthreads();
                b = 0ull;
                for (int j = 0; j < LP_WARPS; ++j) b = warp_best[j] > b ? warp_best[j] : b;
                if (tid == 0) best[r] = b;
                last = b;
                __syncthreads();
            }
        }
    }
    __syncthreads();
    if (slices > 1) {
        cluster_sync();                            // every block's share and list are in place
        if (slice == 0) {
            if (tid == 0) {
                Share b = own_share;
                for (int j = 1; j < slices; ++j) {
                    const unsigned p = cluster_peer(&own_share, (unsigned)j);
                    const Share o = {cluster_f32(p), cluster_f32(p + 4), cluster_f32(p + 8)};
                    b = lp_join(b, o);
                }
                warp_share[0] = b;
            }
            for (int j = tid; j < slices * top; j += LP_THREADS) list[j] = cluster_u64(cluster_peer(&best[j % top], (unsigned)(j / top)));
        }
        cluster_sync();                            // nobody reads this block's memory any more
        if (slice != 0) return;
        const int all = slices * top;
        if (tid < top) groups[tid] = 0ull;         // (there are as many groups as alternatives at most)
        __syncthreads();
        for (int j = tid; j < all; j += LP_THREADS) {
            const Key k = list[j];
            int rank = 0;
            for (int c = 0; c < all; ++c) rank += list[c] > k;
            if (k != 0ull && rank < top) groups[rank] = k;
        }
        __syncthreads();
        if (tid < top) best[tid] = groups[tid];
        if (tid == 0) own_share = warp_share[0];
        __syncthreads();
    }
    // ---- what comes of it
    const Share r = own_share;
    const float ln_s = logf(r.s);
    if (tid == 0) {
        const int token = tokens[row];
        float v = __int_as_float(0x7fc00000);      // NaN: no such token
        if (token < 0 || token >= vocab) {
            if (status) atomicExch(status, 1);
        } else {
            v = (to_f32(x[token]) - r.m) - ln_s;
        }
        logprob[row] = v;
        entropy[row] = ln_s - r.t / r.s * LN2;
    }
    if (tid < top) {
        const Key k = best[tid];
        top_ids[(size_t)row * top + tid] = k == 0ull ? -1 : lp_id(k);
        top_lp[(size_t)row * top + tid] = k == 0ull ? __int_as_float(0x7fc00000) : (lp_logit(k) - r.m) - ln_s;
    }
}

// blocks that share a row: a power of two, while there is at most one a multiprocessor and each has at least 2,048 elements
static int lp_slices(int rows, int vocab) {
    int s = 1;
    while (s < LP_MAX_CLUSTER && 2LL * s * rows <= sm_count() && vocab / (2 * s) >= 2048) s *= 2;
    return s;
}

template <typename T>
static int launch_logprobs(const void* logits, int rows, int vocab, long long stride, const int* tokens, int top, float* logprob, float* entropy,
                           int* top_ids, float* top_lp, int slices, int* status, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long long)rows * slices));
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)slices;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return check_launch("token_logprobs", cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, (const T*)logits, vocab, stride, tokens, top, logprob, entropy,
                                                             top_ids, top_lp, slices, status));
}

// logits [rows] of `vocab`, `stride` elements apart; tokens [rows]; top 0..64 alternatives, at most `vocab`.  slices 0: as many blocks a row as pay.
VAPI_EXPORT int vapi_token_logprobs(const void* logits, int dtype, int rows, int vocab, long long stride, const int* tokens, int top, float* logprob,
                                    float* entropy, int* top_ids, float* top_lp, int slices, int* status, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (vocab <= 0) return fail(-1, "token_logprobs: no tokens in the vocabulary");
    if (top < 0 || top > LP_MAX_TOP || top > vocab) return fail(-1, "token_logprobs: %d alternatives are outside 0..%d, or more than %d tokens", top, LP_MAX_TOP, vocab);
    if (slices < 0 || slices > LP_MAX_CLUSTER || (slices & (slices - 1)) != 0) return fail(-1, "token_logprobs: %d slices are not a power of two up to %d", slices, LP_MAX_CLUSTER);
    if (vocab > 0x7fffffff - 16) return fail(-1, "token_logprobs: a vocabulary of %d is too large", vocab);
    if (slices == 0) slices = lp_slices(rows, vocab);
    if ((long long)rows * slices > 0x7fffffffLL) return fail(-1, "token_logprobs: %d rows exceed the grid", rows);
    if (dtype == VAPI_F32) return launch_logprobs<float>(logits, rows, vocab, stride, tokens, top, logprob, entropy, top_ids, top_lp, slices, status, stream);
    if (dtype == VAPI_BF16) return launch_logprobs<__nv_bfloat16>(logits, rows, vocab, stride, tokens, top, logprob, entropy, top_ids, top_lp, slices, status, stream);
    return fail(-2, "token_logprobs: unsupported dtype %d", dtype);
}

VAPI_EXPORT const char* vapi_last_error() { return error_buffer(); }
