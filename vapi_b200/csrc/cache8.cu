// A paged cache of keys and values in 8 bits: the write that quantises, the read that gives values back, and causal GQA
// attention over it.
//
// A number is code * 2^e: the code is an e4m3 number (four exponent bits, three of the mantissa, largest 448), and every block
// of 16 tokens of a head has one e, for keys and for values apart.  e is the smallest in -110 .. 119 with which the block's
// largest magnitude fits 448.  Powers of two because
//  * multiplying by one is exact, so a code is the same in every arithmetic that rounds to nearest even, and code * 2^e is a
//    bfloat16 number;
//  * a block is written over several steps, and when a later token needs a larger e the older codes move onto it exactly, but
//    for those that fall below the smallest e4m3 numbers (2^-6 of a code; the largest is 448).
// A finer scale would buy nothing: e4m3's rounding is relative to each number, not to the block's largest.
//
// Layout of a layer: codes [pages][2 (k, v)][nkv][page_size][d], e [pages][2][nkv][page_size / 16].  The 16 tokens of a block of
// one head are 16 * d bytes in one piece.
#include "cache8.cuh"
#include "cache8_decode.cuh"
#include "cache8_prompt.cuh"

using namespace vapi;

// ---- the write ----------------------------------------------------------------------------------
// The general kernel: one warp per (token, head) of a fused row [q heads | k heads | v heads]:
//   q: norm (if qw) -> rotation (if cosr) -> q_out;
//   k, v: a warp takes all the step's tokens of its block of 16, if its token is the first of them (slots that follow one
//   another within a block), else it has nothing to do.  First pass: the largest magnitude (k normed, rotated and rounded to the
//   activations' type, as an unquantised cache would hold it).  Then e, the older tokens of the block moved onto it if it
//   grew, and a second pass over the same rows (they are in L1 by then) that writes the codes.
// A new block's first token (place 0) starts its e afresh: what a page held before is never looked at.
constexpr int W8_WARPS = 4;
constexpr int W8_MAX_D = 256;

template <typename T>
__global__ void __launch_bounds__(W8_WARPS * 32)
write8_kernel(const T* __restrict__ qkv, const float* __restrict__ qw, const float* __restrict__ kw, float eps, const float* __restrict__ cosr,
              const float* __restrict__ sinr, int rot, T* __restrict__ q_out, unsigned char* __restrict__ codes, signed char* __restrict__ exps,
              const int* __restrict__ slots, int n, int nh, int nkv, int d, int page_size, int num_pages, int* __restrict__ status) {
    __shared__ float sh[W8_WARPS][W8_MAX_D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads = nh + 2 * nkv;
    const long long item = (long long)blockIdx.x * W8_WARPS + warp;
    pdl_trigger();
    if (item >= (long long)n * heads) {
        pdl_wait();
        return;
    }
    const int t = (int)(item / heads), h = (int)(item - (long long)t * heads);
    const bool is_q = h < nh, is_k = !is_q && h < nh + nkv;
    // (slots are host-copied index data: safe before the wait)
    int slot = 0, count = 1;
    bool mine = true;
    if (!is_q) {
        slot = slots[t];
        const int place = slot & (C8_BLOCK - 1);
        mine = t == 0 || place == 0 || slot < 0 || slots[t - 1] != slot - 1;
        const bool follows = lane < C8_BLOCK && place + lane < C8_BLOCK && t + lane < n && slots[min(t + lane, n - 1)] == slot + lane;
        count = __ffs(~__ballot_sync(0xffffffffu, follows)) - 1;
    }
    pdl_wait();
    if (!mine) return;

    const float* w = is_q ? qw : (is_k ? kw : nullptr);
    const bool rope = (is_q || is_k) && cosr != nullptr;
    const int half = rot >> 1;
    float* s = sh[warp];
    // element i of token t + j, as the activations' type holds it
    auto row = [&](int j) { return qkv + ((size_t)(t + j) * heads + h) * d; };
    auto inv_norm = [&](int j) {
        const T* src = row(j);
        __syncwarp();
        float ss = 0.f;
        for (int i = lane; i < d; i += 32) {
            const float v = to_f32(src[i]);
            s[i] = v;
            ss += v * v;
        }
        __syncwarp();
        return w ? rsqrtf(warp_sum(ss) / (float)d + eps) : 1.f;
    };
    auto element = [&](int j, int i, float inv) {
        float v = w ? s[i] * inv * w[i] : s[i];
        if (rope && i < rot) {
            const int jj = i < half ? i : i - half;
            const int pi = i < half ? i + half : i - half;
            const float pv = w ? s[pi] * inv * w[pi] : s[pi];
            const float c = cosr[(size_t)(t + j) * half + jj], sn = sinr[(size_t)(t + j) * half + jj];
            v = i < half ? v * c - pv * sn : v * c + pv * sn;
        }
        return round_to<T>(v);
    };
    if (is_q) {
        const float inv = inv_norm(0);
        for (int i = lane; i < d; i += 32) q_out[((size_t)t * nh + h) * d + i] = from_f32<T>(element(0, i, inv));
        return;
    }
    const int page = slot / page_size, off = slot - page * page_size, place = off & (C8_BLOCK - 1);
    if (slot < 0 || page >= num_pages) {
        if (lane == 0 && status) atomicExch(status, 2);
        return;
    }
    const int g = is_k ? h - nh : h - nh - nkv;
    const size_t head = ((size_t)page * 2 + (is_k ? 0 : 1)) * nkv + g;
    unsigned char* block = codes + (head * page_size + off - place) * d;
    signed char* exp_at = exps + head * (page_size / C8_BLOCK) + off / C8_BLOCK;

    float amax = 0.f;
    for (int j = 0; j < count; ++j) {
        const float inv = inv_norm(j);
        for (int i = lane; i < d; i += 32) {
            const float a = fabsf(element(j, i, inv));
            if (a < INFINITY) amax = fmaxf(amax, a);              // (false for NaN too)
        }
    }
    int e = c8_exponent(warp_max(amax));
    if (place > 0) {
        const int old = *exp_at;
        e = max(e, old);
        if (e > old) {                                             // the block's older tokens, four codes a lane (d is a multiple of 16)
            unsigned* older = reinterpret_cast<unsigned*>(block);
            const float f = c8_power(max(old - e, -126));          // (2^-126 of any code rounds to zero)
            for (int i = lane; i < place * d / 4; i += 32) older[i] = c8_rescale(older[i], f);
        }
    }
    __syncwarp();                                                  // every lane has read the old e
    if (lane == 0) *exp_at = (signed char)e;
    const float f = c8_power(-e);
    for (int j = 0; j < count; ++j) {
        const float inv = inv_norm(j);
        for (int i = lane; i < d; i += 32) block[(size_t)(place + j) * d + i] = c8_code(element(j, i, inv) * f);
    }
}

// The same for bfloat16, head size 64 or 128 and a rotation over the whole head (or none), with 16-byte accesses and in one pass: D / 16
// lanes take one (token, head), a lane 8 elements of the first half and their partners of the second.  The blocks before `q_blocks`
// take the queries; a warp of the others one head's keys or values of `GROUP` tokens of the step, and of these the runs that begin
// among them: 32 / (D / 16) tokens of a run at a time, all of whose loads are under way together, kept as bfloat16 until
// the block's scale is known.  GROUP 16 for prompts (a run begins in every 16 tokens, but for the ends), 1 for decode steps, where
// each token is a run and 16 of them in a row would be a warp's alone.  Bound by the way of its rows (a chain of slot, row, exponent and, where it
// grew, older codes): 2,048 tokens of 32 / 8 heads of 64 in 7.6 us, 3.1 TB/s of rows, queries and codes, on the general kernel 64; one token 2.5 (3.3).
template <int D>
struct W8Row {                                     // 8 + 8 elements of a (token, head), normed, rotated and rounded
    uint4 lo, hi;
    __device__ __forceinline__ void load(const __nv_bfloat16* src, bool ok, const float* w, float eps, const float* cosr, const float* sinr, int e) {
        constexpr int G = D / 16;
        float a[8], b[8];
        const uint4 ra = ok ? *reinterpret_cast<const uint4*>(src + e) : make_uint4(0u, 0u, 0u, 0u);
        const uint4 rb = ok ? *reinterpret_cast<const uint4*>(src + D / 2 + e) : make_uint4(0u, 0u, 0u, 0u);
        const unsigned wa[4] = {ra.x, ra.y, ra.z, ra.w}, wb[4] = {rb.x, rb.y, rb.z, rb.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[2 * i] = __uint_as_float(wa[i] << 16); a[2 * i + 1] = __uint_as_float(wa[i] & 0xffff0000u);
            b[2 * i] = __uint_as_float(wb[i] << 16); b[2 * i + 1] = __uint_as_float(wb[i] & 0xffff0000u);
        }
        if (w) {                                   // (the same for the whole warp)
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float inv = rsqrtf(ss / (float)D + eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a[i] = a[i] * inv * w[e + i];
                b[i] = b[i] * inv * w[D / 2 + e + i];
            }
        }
        if (cosr && ok) {
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const float4 c = *reinterpret_cast<const float4*>(cosr + e + i), s = *reinterpret_cast<const float4*>(sinr + e + i);
                const float cc[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float x = a[i + k], y = b[i + k];
                    a[i + k] = x * cc[k] - y * sn[k];
                    b[i + k] = y * cc[k] + x * sn[k];
                }
            }
        }
        lo = make_uint4(pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]), pack_bf16(a[4], a[5]), pack_bf16(a[6], a[7]));
        hi = make_uint4(pack_bf16(b[0], b[1]), pack_bf16(b[2], b[3]), pack_bf16(b[4], b[5]), pack_bf16(b[6], b[7]));
    }
    // the largest finite magnitude
    __device__ __forceinline__ float largest() const {
        const unsigned w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = fabsf(__uint_as_float(w[i] << 16)), y = fabsf(__uint_as_float(w[i] & 0xffff0000u));
            m = x < INFINITY ? fmaxf(m, x) : m;
            m = y < INFINITY ? fmaxf(m, y) : m;
        }
        return m;
    }
    static __device__ __forceinline__ uint2 codes(const uint4& v, float f) {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
        unsigned c[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            c[i] = c8_codes4(__uint_as_float(w[2 * i] << 16) * f, __uint_as_float(w[2 * i] & 0xffff0000u) * f, __uint_as_float(w[2 * i + 1] << 16) * f,
                             __uint_as_float(w[2 * i + 1] & 0xffff0000u) * f);
        return make_uint2(c[0], c[1]);
    }
};

template <int D, int GROUP>
__global__ void __launch_bounds__(W8_WARPS * 32)
write8_vec_kernel(const __nv_bfloat16* __restrict__ qkv, const float* __restrict__ qw, const float* __restrict__ kw, float eps, const float* __restrict__ cosr,
                  const float* __restrict__ sinr, __nv_bfloat16* __restrict__ q_out, unsigned char* __restrict__ codes, signed char* __restrict__ exps,
                  const int* __restrict__ slots, int n, int nh, int nkv, int page_size, int num_pages, int q_blocks, int* __restrict__ status) {
    constexpr int G = D / 16, TOKENS = 32 / G, PASSES = C8_BLOCK / TOKENS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane / G, e = lane % G * 8;
    const int heads = nh + 2 * nkv;
    pdl_trigger();
    if ((int)blockIdx.x < q_blocks) {
        pdl_wait();
        const long long item = ((long long)blockIdx.x * W8_WARPS + warp) * TOKENS + part;
        const bool ok = item < (long long)n * nh;
        const int t = ok ? (int)(item / nh) : 0, h = ok ? (int)(item - (long long)t * nh) : 0;
        W8Row<D> r;
        r.load(qkv + ((size_t)t * heads + h) * D, ok, qw, eps, cosr ? cosr + (size_t)t * (D / 2) : nullptr, sinr ? sinr + (size_t)t * (D / 2) : nullptr, e);
        if (ok) {
            __nv_bfloat16* dst = q_out + (size_t)item * D + e;
            *reinterpret_cast<uint4*>(dst) = r.lo;
            *reinterpret_cast<uint4*>(dst + D / 2) = r.hi;
        }
        return;
    }
    const long long item = (long long)(blockIdx.x - q_blocks) * W8_WARPS + warp;
    const int t0 = (int)(item / (2 * nkv)) * GROUP, hk = (int)(item % (2 * nkv));
    if (t0 >= n) {
        pdl_wait();
        return;
    }
    // where runs begin (slots are host-copied index data: safe before the wait)
    const int at = min(t0 + lane, n - 1), mine = slots[at];
    const bool first = lane < GROUP && t0 + lane < n && (at == 0 || (mine & (C8_BLOCK - 1)) == 0 || mine < 0 || slots[at - 1] != mine - 1);
    unsigned runs = __ballot_sync(0xffffffffu, first);
    pdl_wait();
    const bool is_k = hk < nkv;
    const int g = is_k ? hk : hk - nkv;
    for (; runs; runs &= runs - 1) {
        const int j0 = __ffs(runs) - 1, t = t0 + j0, slot = __shfl_sync(0xffffffffu, mine, j0);
        const int page = slot / page_size, off = slot - page * page_size, place = off & (C8_BLOCK - 1);
        const bool follows = lane < C8_BLOCK && place + lane < C8_BLOCK && t + lane < n && slots[min(t + lane, n - 1)] == slot + lane;
        const int count = __ffs(~__ballot_sync(0xffffffffu, follows)) - 1;
        if (slot < 0 || page >= num_pages) {
            if (lane == 0 && status) atomicExch(status, 2);
            continue;
        }
        W8Row<D> r[PASSES];
        float amax = 0.f;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int j = p * TOKENS + part;
            const bool ok = j < count;
            const size_t row = ok ? t + j : t;
            r[p].load(qkv + (row * heads + nh + hk) * D, ok, is_k ? kw : nullptr, eps, is_k && cosr ? cosr + row * (D / 2) : nullptr,
                      is_k && sinr ? sinr + row * (D / 2) : nullptr, e);
            amax = fmaxf(amax, r[p].largest());
        }
        int x = c8_exponent(warp_max(amax));
        const size_t head = ((size_t)page * 2 + (is_k ? 0 : 1)) * nkv + g;
        unsigned char* block = codes + (head * page_size + off - place) * D;
        signed char* exp_at = exps + head * (page_size / C8_BLOCK) + off / C8_BLOCK;
        if (place > 0) {
            const int old = *exp_at;
            x = max(x, old);
            if (x > old) {                                         // the block's older tokens
                unsigned* older = reinterpret_cast<unsigned*>(block);
                const float f = c8_power(max(old - x, -126));
                for (int i = lane; i < place * D / 4; i += 32) older[i] = c8_rescale(older[i], f);
            }
        }
        __syncwarp();                                              // every lane has read the old exponent
        if (lane == 0) *exp_at = (signed char)x;
        const float f = c8_power(-x);
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int j = p * TOKENS + part;
            if (j >= count) continue;
            unsigned char* dst = block + (place + j) * D + e;
            *reinterpret_cast<uint2*>(dst) = W8Row<D>::codes(r[p].lo, f);
            *reinterpret_cast<uint2*>(dst + D / 2) = W8Row<D>::codes(r[p].hi, f);
        }
    }
}

// Tokens of a step from which on a warp takes 16 of them: steps as large are a portion's.  (Single tokens beside it then take turns in a warp; the rule goes by
// the step and not by its runs.)  us of one and of 16 a warp, 32 / 8 heads of 64: runs of
// 128 tokens 3.3 / 3.2, 256 3.9 / 3.5, 512 5.4 / 3.8, 2,048 14.6 / 7.6; single tokens, 8 of them 2.8 / 14.3, 64 3.4 / 28.6.
constexpr int W8_GROUP_TOKENS = 512;

template <int D>
static int launch_write8_vec(const void* qkv, const float* qw, const float* kw, float eps, const float* cosr, const float* sinr, void* q_out, void* codes, void* exps,
                             const int* slots, int n, int nh, int nkv, int page_size, int num_pages, int* status, cudaStream_t stream) {
    const int group = n >= W8_GROUP_TOKENS ? C8_BLOCK : 1;
    const long long per = (long long)W8_WARPS * (32 / (D / 16)), q_blocks = ((long long)n * nh + per - 1) / per;
    const long long blocks = q_blocks + ((long long)((n + group - 1) / group) * 2 * nkv + W8_WARPS - 1) / W8_WARPS;
    if (blocks > 0x7fffffffLL) return fail(-1, "qk_norm_rope_write8: %d tokens exceed the grid", n);
    return check_launch("qk_norm_rope_write8", launch(group == 1 ? write8_vec_kernel<D, 1> : write8_vec_kernel<D, C8_BLOCK>, (unsigned)blocks, W8_WARPS * 32, 0, stream,
                                                      (const __nv_bfloat16*)qkv, qw, kw, eps, cosr, sinr, (__nv_bfloat16*)q_out, (unsigned char*)codes,
                                                      (signed char*)exps, slots, n, nh, nkv, page_size, num_pages, (int)q_blocks, status));
}

VAPI_EXPORT int vapi_qk_norm_rope_write8(const void* qkv, int dtype, const float* qw, const float* kw, float eps, const float* cosr,
                                         const float* sinr, int rot, void* q_out, void* codes, void* exps, const int* slots, int n,
                                         int nh, int nkv, int d, int page_size, int num_pages, int* status, cudaStream_t stream) {
    if (n <= 0) return 0;
    if (d < 16 || d > W8_MAX_D || d % 16 != 0) return fail(-1, "qk_norm_rope_write8: head_dim %d is not a multiple of 16 in 16..256", d);
    if (nh <= 0 || nkv <= 0) return fail(-1, "qk_norm_rope_write8: no heads");
    if (cosr && (rot <= 0 || rot > d || rot % 2 != 0)) return fail(-1, "qk_norm_rope_write8: rotation width %d does not fit head_dim %d", rot, d);
    if (page_size <= 0 || page_size % C8_BLOCK != 0 || num_pages <= 0) return fail(-1, "qk_norm_rope_write8: page size %d is not a multiple of 16, or there are no pages", page_size);
    // (older codes of a block are read by words; the read and attention take pieces of 16 bytes)
    if (((uintptr_t)codes & 15) != 0) return fail(-1, "qk_norm_rope_write8: the codes are not 16-byte aligned");
    // (16-byte rows of everything that is read or written by the piece)
    if (dtype == VAPI_BF16 && (d == 64 || d == 128) && (!cosr || rot == d) &&
        (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)codes | (uintptr_t)cosr | (uintptr_t)sinr) & 15) == 0)
        return d == 64 ? launch_write8_vec<64>(qkv, qw, kw, eps, cosr, sinr, q_out, codes, exps, slots, n, nh, nkv, page_size, num_pages, status, stream)
                       : launch_write8_vec<128>(qkv, qw, kw, eps, cosr, sinr, q_out, codes, exps, slots, n, nh, nkv, page_size, num_pages, status, stream);
    const long long blocks = ((long long)n * (nh + 2 * nkv) + W8_WARPS - 1) / W8_WARPS;
    if (blocks > 0x7fffffffLL) return fail(-1, "qk_norm_rope_write8: %d tokens exceed the grid", n);
    cudaError_t e;
    if (dtype == VAPI_F32)
        e = launch(write8_kernel<float>, (unsigned)blocks, W8_WARPS * 32, 0, stream, (const float*)qkv, qw, kw, eps, cosr, sinr, rot, (float*)q_out,
                   (unsigned char*)codes, (signed char*)exps, slots, n, nh, nkv, d, page_size, num_pages, status);
    else if (dtype == VAPI_BF16)
        e = launch(write8_kernel<__nv_bfloat16>, (unsigned)blocks, W8_WARPS * 32, 0, stream, (const __nv_bfloat16*)qkv, qw, kw, eps, cosr, sinr, rot,
                   (__nv_bfloat16*)q_out, (unsigned char*)codes, (signed char*)exps, slots, n, nh, nkv, d, page_size, num_pages, status);
    else
        return fail(-2, "qk_norm_rope_write8: unsupported dtype %d", dtype);
    return check_launch("qk_norm_rope_write8", e);
}

// ---- the read -----------------------------------------------------------------------------------
// Whole pages as numbers, in the order of `pages`: 16 codes (one 16-byte load) a thread; a page id outside the pool leaves zeros
// and a status.  32 pages of 64 tokens, 8 heads of 64, 3.0 us: a launch and one way to memory and back.
template <typename T>
__global__ void read8_kernel(const unsigned char* __restrict__ codes, const signed char* __restrict__ exps, const int* __restrict__ pages,
                             T* __restrict__ out, long long pieces, int per_page, int per_block, int num_pages, int* __restrict__ status) {
    pdl_trigger();
    pdl_wait();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= pieces) return;
    const int at = (int)(i / per_page), piece = (int)(i - (long long)at * per_page);
    const int page = pages[at];
    float v[16];
    if (page < 0 || page >= num_pages) {
        if (piece == 0 && status) atomicExch(status, 4);
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = 0.f;
    } else {
        const uint4 c = reinterpret_cast<const uint4*>(codes)[(size_t)page * per_page + piece];
        const float f = c8_power(exps[(size_t)page * (per_page / per_block) + piece / per_block]);
        const unsigned w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4 x = c8_floats(w[k]);
            v[4 * k] = x.x * f; v[4 * k + 1] = x.y * f; v[4 * k + 2] = x.z * f; v[4 * k + 3] = x.w * f;
        }
    }
    T* dst = out + 16 * i;
    if (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) reinterpret_cast<float4*>(dst)[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    } else {
        unsigned w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
            w[k] = *reinterpret_cast<const unsigned*>(&b);
        }
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

VAPI_EXPORT int vapi_cache8_read(const void* codes, const void* exps, const int* pages, void* out, int dtype, int count, int nkv, int d,
                                 int page_size, int num_pages, int* status, cudaStream_t stream) {
    if (count <= 0) return 0;
    if (d < 16 || d > 256 || d % 16 != 0) return fail(-1, "cache8_read: head_dim %d is not a multiple of 16 in 16..256", d);
    if (nkv <= 0 || page_size <= 0 || page_size % C8_BLOCK != 0 || num_pages <= 0) return fail(-1, "cache8_read: page size %d is not a multiple of 16, or there are no pages", page_size);
    if (((uintptr_t)codes & 15) != 0 || ((uintptr_t)out & 15) != 0) return fail(-1, "cache8_read: the codes or the output are not 16-byte aligned");
    const long long per_page = 2LL * nkv * page_size * (d / 16), pieces = per_page * count;
    if (per_page > 0x7fffffffLL || (pieces + 255) / 256 > 0x7fffffffLL) return fail(-1, "cache8_read: %d pages exceed the grid", count);
    const unsigned blocks = (unsigned)((pieces + 255) / 256);
    cudaError_t e;
    if (dtype == VAPI_F32)
        e = launch(read8_kernel<float>, blocks, 256, 0, stream, (const unsigned char*)codes, (const signed char*)exps, pages, (float*)out, pieces,
                   (int)per_page, d, num_pages, status);
    else if (dtype == VAPI_BF16)
        e = launch(read8_kernel<__nv_bfloat16>, blocks, 256, 0, stream, (const unsigned char*)codes, (const signed char*)exps, pages, (__nv_bfloat16*)out,
                   pieces, (int)per_page, d, num_pages, status);
    else
        return fail(-2, "cache8_read: unsupported dtype %d", dtype);
    return check_launch("cache8_read", e);
}

// ---- attention: the general kernel --------------------------------------------------------------
// float32 activations, head sizes other than 64 and 128, queries at any alignment; float FMAs.  A block owns R rows (query token, q head of the group) of
// one (sequence, kv head); its eight warps, and those of the up to 8 blocks of its cluster, each take a run of the key tiles, 32 keys a tile,
// a lane one key of the scores (a code is turned once for all rows) and every 32nd element of the output.  One pass with a running maximum and sum a
// row, in float; the results are joined in the order of warps, then of blocks.  Bound by its loads of single codes and float operations.  32 / 8 heads
// of 64, float32: one request of 4,090 keys 32 us, 64 of 128 to 2,048 146, 8 of 32,000 700 (in bfloat16 the mma.sync kernel takes 6, 20 and 48), 500 tokens
// behind 100 245 (15).
constexpr int G8_KEYS = 32, G8_WARPS = 8, G8_MAX_CLUSTER = 8;

template <typename T, int DMAX, int R>
__global__ void __launch_bounds__(G8_WARPS * 32)
attention8_kernel(const C8Params p, const T* __restrict__ q, T* __restrict__ out, const int splits) {
    constexpr int C = DMAX / 32;
    extern __shared__ __align__(16) float g8_smem[];
    __shared__ float sM[G8_WARPS][R], sL[G8_WARPS][R], xM[R], xL[R];
    const int d = p.d, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* sQ = g8_smem;                                            // [R][d]; then, in its place, the block's O
    float* sO = g8_smem + R * d;                                    // [warp][R][d]
    const int rank = (int)blockIdx.x % splits, s = blockIdx.z, g = blockIdx.y, n_rep = p.nh / p.nkv;
    pdl_trigger();
    pdl_wait();
    const int q0 = p.cu_q[s], qlen = p.cu_q[s + 1] - q0, klen = p.seqlens_k[s];
    const int rows_total = qlen * n_rep, r0 = (int)blockIdx.x / splits * R;
    if (r0 >= rows_total) return;                                   // (the same for the whole cluster)
    const int base = klen - qlen;
    const int p_min = base + r0 / n_rep, p_max = base + (min(rows_total, r0 + R) - 1) / n_rep;
    const int lo = p.window > 0 ? max(0, p_min - p.window + 1) : 0;
    for (int i = threadIdx.x; i < R * d; i += blockDim.x) {
        const int r = i / d, c = i - r * d, rr = r0 + r, tok = rr / n_rep;
        sQ[i] = rr < rows_total ? to_f32(q[(size_t)(q0 + tok) * p.q_row_stride + (size_t)(g * n_rep + rr - tok * n_rep) * d + c]) * p.scale_log2e : 0.f;
    }
    int pos[R];                                                     // -1: sees nothing
    float m[R], l[R], o[R][C];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        pos[r] = r0 + r < rows_total ? base + (r0 + r) / n_rep : -1;
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) o[r][c] = 0.f;
    }
    __syncthreads();
    const int* bt = p.block_table + (size_t)s * p.table_stride;
    const int t_lo = lo / G8_KEYS, unit = rank * G8_WARPS + warp, units = splits * G8_WARPS;
    const long long tiles = p_max < lo ? 0 : p_max / G8_KEYS - t_lo + 1;
    for (int t = t_lo + (int)(tiles * unit / units); t < t_lo + (int)(tiles * (unit + 1) / units); ++t) {
        const int key = t * G8_KEYS + lane;
        const bool there = key >= lo && key <= p_max;               // (keys that no row sees may hold anything, and are not read)
        int page = there ? bt[key / p.page_size] : -1;
        if (there && (page < 0 || page >= p.num_pages) && p.status) atomicExch(p.status, 4);
        if (page >= p.num_pages) page = -1;
        const int off = key % p.page_size;
        const size_t head = ((size_t)max(page, 0) * 2) * p.nkv + g;
        float x[R];
#pragma unroll
        for (int r = 0; r < R; ++r) x[r] = 0.f;
        float fk = 0.f, fv = 0.f;                                   // (a page that is none: zeros)
        if (page >= 0) {
            const size_t e = head * (p.page_size / C8_BLOCK) + off / C8_BLOCK;
            fk = c8_power(p.exps[e]);
            fv = c8_power(p.exps[e + (size_t)p.nkv * (p.page_size / C8_BLOCK)]);
            const uint4* k = reinterpret_cast<const uint4*>(p.codes + (head * p.page_size + off) * d);
            for (int c = 0; c < d / 16; ++c) {
                const uint4 v = k[c];
                const float4 a[4] = {c8_floats(v.x), c8_floats(v.y), c8_floats(v.z), c8_floats(v.w)};
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 b = *reinterpret_cast<const float4*>(sQ + r * d + 16 * c + 4 * i);
                        x[r] = fmaf(a[i].x, b.x, fmaf(a[i].y, b.y, fmaf(a[i].z, b.z, fmaf(a[i].w, b.w, x[r]))));
                    }
            }
        }
        unsigned seen[R], all = 0xffffffffu, any = 0u;              // keys of the tile that a row sees
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool sees = there && key <= pos[r] && (p.window <= 0 || key > pos[r] - p.window);
            seen[r] = __ballot_sync(0xffffffffu, sees);
            x[r] = sees ? x[r] * fk : -INFINITY;
            any |= seen[r];
            if (r0 + r < rows_total) all &= seen[r];
            if (!seen[r]) { x[r] = 0.f; continue; }
            const float mx = fmaxf(m[r], warp_max(x[r])), use = mx == -INFINITY ? 0.f : mx;
            const float alpha = exp2f(m[r] - use);
            x[r] = sees ? exp2f(x[r] - use) : 0.f;                  // the weight
            m[r] = mx;
            l[r] = l[r] * alpha + x[r];                             // (a lane's share of the sum)
#pragma unroll
            for (int c = 0; c < C; ++c) o[r][c] *= alpha;
        }
#pragma unroll 4
        for (int k = 0; k < G8_KEYS; ++k) {
            if (!(any >> k & 1)) continue;
            const int page_k = __shfl_sync(0xffffffffu, page, k);
            const float f = __shfl_sync(0xffffffffu, fv, k);
            const unsigned char* src = p.codes + ((((size_t)max(page_k, 0) * 2 + 1) * p.nkv + g) * p.page_size + (t * G8_KEYS + k) % p.page_size) * d;
            float v[C];
#pragma unroll
            for (int c = 0; c < C; ++c) v[c] = page_k >= 0 && c * 32 + lane < d ? c8_floats(src[c * 32 + lane]).x * f : 0.f;
            const bool every = all >> k & 1;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float w = __shfl_sync(0xffffffffu, x[r], k);
                if (!every && !(seen[r] >> k & 1)) continue;        // (a NaN that a row does not see stays where it is)
#pragma unroll
                for (int c = 0; c < C; ++c) o[r][c] = fmaf(w, v[c], o[r][c]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float sum = warp_sum(l[r]);
        if (lane == 0) { sM[warp][r] = m[r]; sL[warp][r] = sum; }
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (c * 32 + lane < d) sO[(warp * R + r) * d + c * 32 + lane] = o[r][c];
    }
    __syncthreads();
    auto store = [&](int r, int c, float v, float sum) {
        const int rr = r0 + r, tok = rr / n_rep;
        if (rr >= rows_total) return;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;             // a row that sees nothing: zeros
        out[((size_t)(q0 + tok) * p.nh + g * n_rep + rr - tok * n_rep) * d + c] = from_f32<T>(v * inv);
    };
    for (int i = threadIdx.x; i < R * d; i += G8_WARPS * 32) {
        const int r = i / d, c = i - r * d;
        float mx = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < G8_WARPS; ++w) mx = fmaxf(mx, sM[w][r]);
        const float use = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int w = 0; w < G8_WARPS; ++w) {
            const float f = exp2f(sM[w][r] - use);
            sum = fmaf(sL[w][r], f, sum);
            v = fmaf(sO[(w * R + r) * d + c], f, v);
        }
        if (splits == 1) {
            store(r, c, v, sum);
        } else {
            sQ[i] = v;
            if (c == 0) { xM[r] = mx; xL[r] = sum; }
        }
    }
    if (splits > 1) {
        cluster_sync();                                             // every block's result is in place
        const int mine = (R * d + splits - 1) / splits;
        for (int i = rank * mine + threadIdx.x; i < min((rank + 1) * mine, R * d); i += G8_WARPS * 32) {
            const int r = i / d, c = i - r * d;
            float ms[G8_MAX_CLUSTER], ls[G8_MAX_CLUSTER], vs[G8_MAX_CLUSTER], mx = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
            for (int j = 0; j < G8_MAX_CLUSTER; ++j) {              // (all under way together)
                ms[j] = j < splits ? cluster_f32(cluster_peer(&xM[r], (unsigned)j)) : -INFINITY;
                ls[j] = j < splits ? cluster_f32(cluster_peer(&xL[r], (unsigned)j)) : 0.f;
                vs[j] = j < splits ? cluster_f32(cluster_peer(&sQ[i], (unsigned)j)) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < G8_MAX_CLUSTER; ++j) mx = fmaxf(mx, ms[j]);
            const float use = mx == -INFINITY ? 0.f : mx;
#pragma unroll
            for (int j = 0; j < G8_MAX_CLUSTER; ++j) {
                const float f = exp2f(ms[j] - use);
                sum = fmaf(ls[j], f, sum);
                v = fmaf(vs[j], f, v);
            }
            store(r, c, v, sum);
        }
        cluster_sync();                                             // nobody reads this block's memory any more
    }
}

template <typename T, int DMAX, int R>
static int launch_attention8_of(const C8Params& p, const void* q, void* out, int num_seqs, int max_q, int max_k, int splits, cudaStream_t stream) {
    const long long tiles = ((long long)max_q * (p.nh / p.nkv) + R - 1) / R;
    if (tiles * G8_MAX_CLUSTER > 0x7fffffffLL || p.nkv > 65535 || num_seqs > 65535)
        return fail(-1, "paged_attention8: the step exceeds the grid (%lld row tiles, %d kv heads, %d sequences)", tiles, p.nkv, num_seqs);
    if (splits <= 0) {
        // blocks to two a multiprocessor, while every warp has a tile
        splits = 1;
        while (splits < G8_MAX_CLUSTER && 2 * splits * tiles * p.nkv * num_seqs <= 2LL * sm_count() && 2LL * splits * G8_WARPS * G8_KEYS <= max_k) splits *= 2;
    }
    if (splits > G8_MAX_CLUSTER) splits = G8_MAX_CLUSTER;
    const size_t smem = (size_t)(1 + G8_WARPS) * R * p.d * sizeof(float);
    constexpr size_t most = (size_t)(1 + G8_WARPS) * R * DMAX * sizeof(float);
    auto kern = attention8_kernel<T, DMAX, R>;
    // (the limit of the largest head size, once a device: a limit by the call's would be lowered between another thread's setting and its launch)
    static int ready[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(-101, "paged_attention8: cannot tell the current device");
    if (!ready[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (e != cudaSuccess) return fail(-101, "paged_attention8: cannot reserve %zu bytes of shared memory: %s", most, cudaGetErrorString(e));
        ready[dev] = 1;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * splits), p.nkv, num_seqs);
    cfg.blockDim = dim3(G8_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return check_launch("paged_attention8", cudaLaunchKernelEx(&cfg, kern, p, (const T*)q, (T*)out, splits));
}
template <typename T, int DMAX>
static int launch_attention8(const C8Params& p, const void* q, void* out, int num_seqs, int max_q, int max_k, int splits, cudaStream_t stream) {
    if ((long long)max_q * (p.nh / p.nkv) <= 4) return launch_attention8_of<T, DMAX, 4>(p, q, out, num_seqs, max_q, max_k, splits, stream);
    return launch_attention8_of<T, DMAX, 8>(p, q, out, num_seqs, max_q, max_k, splits, stream);
}

// How many blocks of the mma.sync kernel share the keys of one (sequence, kv head, tile of rows): a power of two up to a cluster's 16, while all
// blocks are on the device at once and each of a block's eight warps still has two blocks of 16 tokens.
static int c8_splits(int num_seqs, int max_q, int max_k, int nh, int nkv, int d) {
    if (num_seqs <= 0 || max_q <= 0 || nkv <= 0) return 1;
    const long long rows = (long long)max_q * (nh / nkv), blocks = (long long)num_seqs * nkv * ((rows + (rows <= 8 ? 7 : 15)) / (rows <= 8 ? 8 : 16));
    const long long slots = d == 64 ? decode8_slots<64>() : decode8_slots<128>();
    int splits = 1;
    while (splits < D8_MAX_CLUSTER && 2 * splits * blocks <= slots && 2LL * splits * 256 <= max_k) splits *= 2;
    return splits;
}

// Whether a step's portions are for the tcgen05 kernel: whether by these estimates it takes less time.  The mma.sync kernel's are rounds of
// blocks of 16 rows, of 5 us and 7.5 (head size 128: 6.5) a thousand keys.  Its tiles are smaller and its keys can be shared out further, so it is
// ahead where rows or keys are few: 32 / 8 heads of 64, us on mma.sync and on tcgen05: 32 tokens of 4,000 15 / 19, 64 22 / 22, 128 35 / 28, 256
// 68 / 30, 2,048 of 8,000 782 / 238; 64 of 32,000 127 / 83; 128 of 1,000 13 / 16; 512 of 512 29 / 14.
template <int HD>
static bool c8_portions_of(const C8Params& p, int n, int num_seqs, int max_q, int max_k) {
    float tcgen05;
    p8_step<HD>(p, n, max_k, tcgen05);
    const long long seen = p.window > 0 && p.window + 16 < max_k ? p.window + 16 : max_k;
    const float blocks = (float)(((long long)n * (p.nh / p.nkv) + 15) / 16 * p.nkv), slots = (float)decode8_slots<HD>();
    const int splits = c8_splits(num_seqs, max_q, max_k, p.nh, p.nkv, HD);
    const float rounds = blocks * splits / slots;
    return tcgen05 < (rounds > 1.f ? rounds : 1.f) * (5.f + (HD == 64 ? 0.0075f : 0.0065f) * (float)seen / (float)splits);
}
static bool c8_portions(const C8Params& p, int n, int num_seqs, int max_q, int max_k) {
    if (max_q < P8_MIN_Q) return false;
    return p.d == 64 ? c8_portions_of<64>(p, n, num_seqs, max_q, max_k) : c8_portions_of<128>(p, n, num_seqs, max_q, max_k);
}

// q: [n, *] with `q_row_stride` elements between tokens, head h at h * d; out: [n, nh * d].
// impl: 0 = the fastest kernel that applies: for bfloat16 and head size 64 or 128 the tcgen05 kernel for steps with a long enough portion
// (c8_portions; in a step of several sequences for those of at least P8_MIN_Q tokens, beside the mma.sync kernel for the others), else the mma.sync
// kernel; the general kernel for everything else.  1 = the general kernel; 2 = the mma.sync kernel, or an error;
// 3 = the tcgen05 kernel for every sequence, or an error.  splits 0: as many as pay (max_k: the most keys
// a sequence has); else those of the mma.sync kernel, up to 16, and at most 8, a power of two, of the tcgen05 kernel.
// settled: no kernel that may still run when this one begins (the one before it, and those that it begins before the end of) writes keys before a sequence's
// own tokens, as in an engine's step; else no key is read before every earlier kernel has ended.  us of one call after another, settled and not, 32 / 8
// heads of 64, over one cache: one request of 4,090 keys 5.9 / 6.2, 64 of 128 to 2,048 19.6 / 20.7, 8 of 32,000 47.0 / 48.8, 2,048 tokens behind 5,952
// 235.7 / 235.7; over three caches in turn 6.5 / 7.1, 20.3 / 21.7 (22.9 without asking for the first chunks ahead of the wait), 51.6 / 52.8, 236.1 / 235.5.
VAPI_EXPORT int vapi_paged_attention8(const void* q, long long q_row_stride, const void* codes, const void* exps, int dtype, const int* block_table,
                                      int table_stride, const int* cu_q, const int* seqlens_k, void* out, int n, int num_seqs, int max_q,
                                      int max_k, int nh, int nkv, int d, int page_size, int num_pages, float scale, int window, int splits,
                                      int impl, int settled, int* status, cudaStream_t stream) {
    if (n <= 0 || num_seqs <= 0 || max_q <= 0) return 0;
    if (d < 16 || d > 256 || d % 16 != 0) return fail(-1, "paged_attention8: head_dim %d is not a multiple of 16 in 16..256", d);
    if (nh <= 0 || nkv <= 0 || nh % nkv != 0) return fail(-1, "paged_attention8: %d heads are not a multiple of %d kv heads", nh, nkv);
    if (page_size <= 0 || page_size % C8_BLOCK != 0 || num_pages <= 0)
        return fail(-1, "paged_attention8: page size %d is not a multiple of 16, or there are no pages", page_size);
    if (((uintptr_t)codes & 15) != 0) return fail(-1, "paged_attention8: the codes are not 16-byte aligned");
    C8Params p;
    p.q_row_stride = q_row_stride; p.codes = (const unsigned char*)codes; p.exps = (const signed char*)exps; p.block_table = block_table;
    p.table_stride = table_stride; p.cu_q = cu_q; p.seqlens_k = seqlens_k; p.nh = nh; p.nkv = nkv; p.d = d; p.page_size = page_size;
    p.num_pages = num_pages; p.scale_log2e = scale * 1.4426950408889634f; p.window = window; p.settled = settled; p.status = status;
    const bool fast = dtype == VAPI_BF16 && (d == 64 || d == 128) && q_row_stride % 8 == 0 && ((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0;
    if (impl >= 2 && (!fast || (impl == 3 && !(scale > 0.f))))
        return fail(-3, "paged_attention8: the tensor-core kernels need bfloat16, head_dim 64 or 128, 16-byte aligned rows and, for portions, a "
                        "positive scale (got dtype %d, head_dim %d, scale %g)", dtype, d, (double)scale);
    if (fast && impl != 1) {
        if ((long long)num_pages * 2 * nkv * (page_size / C8_BLOCK) > 0x7fffffffLL)
            return fail(-1, "paged_attention8: %d pages of %d tokens and %d kv heads are more blocks than an index holds", num_pages, page_size, nkv);
        int rc = 0, most_q = 0x7fffffff;
        if (impl == 3 || (impl == 0 && scale > 0.f && c8_portions(p, n, num_seqs, max_q, max_k))) {
            const int min_q = impl == 3 || num_seqs == 1 ? 1 : P8_MIN_Q;
            rc = d == 64 ? launch_prompt8<64>(p, q, out, n, num_seqs, max_q, max_k, min_q, splits, stream) : launch_prompt8<128>(p, q, out, n, num_seqs, max_q, max_k, min_q, splits, stream);
            if (rc != 0 || min_q == 1) return rc;
            most_q = min_q - 1;
        }
        if (splits <= 0) splits = c8_splits(num_seqs, most_q < max_q ? 1 : max_q, max_k, nh, nkv, d);      // (beside a portion: as for single tokens)
        return d == 64 ? launch_decode8<64>(p, q, out, num_seqs, max_q, max_k, splits, most_q, stream)
                       : launch_decode8<128>(p, q, out, num_seqs, max_q, max_k, splits, most_q, stream);
    }
#define VAPI_ATT8(T, DM) return launch_attention8<T, DM>(p, q, out, num_seqs, max_q, max_k, splits, stream)
    if (dtype == VAPI_F32) {
        if (d <= 64) VAPI_ATT8(float, 64); else if (d <= 128) VAPI_ATT8(float, 128); else VAPI_ATT8(float, 256);
    }
    if (dtype == VAPI_BF16) {
        if (d <= 64) VAPI_ATT8(__nv_bfloat16, 64); else if (d <= 128) VAPI_ATT8(__nv_bfloat16, 128); else VAPI_ATT8(__nv_bfloat16, 256);
    }
#undef VAPI_ATT8
    return fail(-2, "paged_attention8: unsupported dtype %d", dtype);
}

VAPI_EXPORT int vapi_attention8_splits(int num_seqs, int max_q, int max_k, int nh, int nkv, int d) { return c8_splits(num_seqs, max_q, max_k, nh, nkv, d); }
// how many kernels a step of several sequences takes: 2 where its portions go to the tcgen05 kernel and the rest to the mma.sync one
VAPI_EXPORT int vapi_attention8_kernels(int n, int num_seqs, int max_q, int max_k, int nh, int nkv, int d, int window) {
    if (num_seqs <= 1 || nh <= 0 || nkv <= 0 || nh % nkv != 0 || (d != 64 && d != 128)) return 1;
    C8Params p = {};
    p.nh = nh; p.nkv = nkv; p.d = d; p.window = window;
    return c8_portions(p, n, num_seqs, max_q, max_k) ? 2 : 1;
}
VAPI_EXPORT const char* vapi_last_error() { return error_buffer(); }
