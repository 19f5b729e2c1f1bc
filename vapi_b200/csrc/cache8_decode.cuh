// Attention over an 8-bit cache on the tensor cores (mma.sync m16n8k16, f16 in, float accumulate): bfloat16 queries, head size 64
// or 128, any page size and any number of rows.
//
// A decode step reads every key and value of every live request once, so the kernel is built around that stream.  A cluster of
// up to 16 blocks owns one (sequence, kv head, tile of 8 or 16 rows) and its eight (or four) warps each a run of chunks: the 16
// tokens that share a scale, one piece of memory of 16 * head size bytes for K and one for V.  A warp brings its own chunks,
// two at a time, in by bulk copies through a ring of its own, and no warp waits for another before the end, where their partial
// results are joined: through shared memory in a block, through the cluster's among its blocks, always in the same order.
//
//   S^T = K Q^T  16 tokens are a product's rows and 8 query rows its columns, so that four query heads a kv head leave half of it
//                unused and not three quarters.  A code is an f16 number exactly.  A row of Q is scaled by a power of two so that
//                its largest element is near 2^14: f16 then has three bits more than bfloat16 for it, and elements keep all of
//                theirs down to 2^-28 of the largest.  A lane's 16 contiguous bytes of a key are its operands of four k-steps: the
//                order of the head's elements in the sum is free as long as Q follows it, and so no byte moves between lanes.
//   O^T += V^T P^T   P = 2^(s + e - M) with the values' scale 2^e in the exponent and M the largest s + e so far: the product of P and
//                the codes is added up in the tensor core's accumulator as it is.  (One maximum for both would lose, in f16, what a
//                block of large values says at a small weight, or the other way round.)  The sum of weights is taken of 2^(s - m), m
//                the largest s so far.  m and M are only raised when a score passes them by more than 2^8 (f16 holds P up
//                to 2^15, float the sums), which no lane has to ask its neighbours for: a vote a chunk, and a reduction a few times
//                a row.  P is turned about by movmatrix; the values of two tokens are paired by byte permutes.
//
// What bounds it: memory where keys are many (32 / 8 heads of 64, 8 requests of 32,000 keys 47 us, 5.6 TB/s; the 16-bit kernel 85), the integer
// operations that turn codes to halves close behind; for one request of 4,090 keys (6.0 us) the way of table, exponents and codes after one another.
//
// Keys that a row does not see are masked by selection, and the values of those that no row of the block sees taken as zeros.  (A NaN among the
// values that some of the block's rows see and others do not can reach the others through 0 * NaN; the step that wrote it was lost.)
#pragma once
#include "cache8.cuh"
#include "cluster.cuh"
#include "tcgen05.cuh"           // mbarriers with bounded waits

namespace vapi {

constexpr int D8_WARPS = 8, D8_FEW_WARPS = 4;                                           // of a block; of one where blocks are many and keys few
constexpr int D8_MAX_CLUSTER = 16;
constexpr int D8_STAGES = 3;                                                           // of two chunks of K and of V
constexpr float D8_RAISE = 8.f;                                                        // log2 units by which a score must pass a maximum to raise it
template <int HD> constexpr int D8_CHUNK = C8_BLOCK * HD;                              // bytes of a chunk of K, or of V
template <int HD> constexpr int D8_WARP_BYTES = D8_STAGES * 4 * D8_CHUNK<HD>;
template <int HD, int WARPS> constexpr size_t D8_SMEM = (size_t)WARPS * D8_WARP_BYTES<HD>;

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit numbers, a row's pair of columns a lane, about its diagonal
__device__ __forceinline__ unsigned d8_turned(unsigned x) {
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ unsigned d8_half2(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float d8_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void d8_copy(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void d8_prefetch(const void* src, unsigned bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 d8_lds16(unsigned addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 d8_lds8(unsigned addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
template <int V> struct Number { static constexpr int value = V; };

// WIDE: tiles of 16 rows, else of 8.
template <int HD, bool WIDE, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, (HD == 64 ? 16 : 8) / WARPS)
decode8_kernel(const C8Params p, const __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ out, const int splits, const int most_q) {
    constexpr int ROWS = WIDE ? 16 : 8, H = WIDE ? 2 : 1, CHUNK = D8_CHUNK<HD>;
    constexpr int KS = HD / 16, Q64 = HD / 64, VW = HD / 32;                // k-steps of S; runs of 64 elements; words of a token's values that a lane holds
    extern __shared__ __align__(128) unsigned char d8_smem[];
    __shared__ __align__(8) unsigned long long bars[WARPS * D8_STAGES];
    __shared__ float sM[WARPS][ROWS], sR[WARPS][ROWS], sL[WARPS][ROWS];
    __shared__ float xM[ROWS], xR[ROWS], xL[ROWS];
    __shared__ __align__(16) float xO[ROWS][HD];
    __shared__ int failed;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
    const int rank = (int)blockIdx.x % splits, tile = (int)blockIdx.x / splits, g = blockIdx.y, s = blockIdx.z;
    pdl_trigger();
    // index data was copied from the host before the step's first kernel: safe before the wait
    const int q0 = p.cu_q[s], qlen = p.cu_q[s + 1] - q0, klen = p.seqlens_k[s];
    const int n_rep = p.nh / p.nkv, rows_total = qlen * n_rep, r0 = tile * ROWS;
    if (r0 >= rows_total || qlen > most_q) {                                // longer portions are another kernel's (the same for the whole cluster)
        pdl_wait();
        return;
    }
    const int base = klen - qlen;
    const int p_min = base + r0 / n_rep, p_max = base + (min(rows_total, r0 + ROWS) - 1) / n_rep;
    const int key_lo = p.window > 0 ? max(0, p_min - p.window + 1) : 0;
    const int c_lo = key_lo / C8_BLOCK;
    const long long chunks = p_max < key_lo ? 0 : p_max / C8_BLOCK - c_lo + 1;
    const int units = splits * WARPS, unit = rank * WARPS + warp;
    const int begin = c_lo + (int)(chunks * unit / units), end = c_lo + (int)(chunks * (unit + 1) / units), nt = end - begin, pairs = (nt + 1) / 2;

    const unsigned bar = smem_u32(bars + warp * D8_STAGES), ring = smem_u32(d8_smem + (size_t)warp * D8_WARP_BYTES<HD>);
    if (lane == 0) {
        for (int i = 0; i < D8_STAGES; ++i) mbar_init(bar + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 0) failed = 0;
    __syncthreads();

    // Where 32 chunks at a time lie, one a lane, and their scales: looked up as the copies reach them, used as the products do.
    const int* bt = p.block_table + (size_t)s * p.table_stride;
    const int per_head = p.page_size / C8_BLOCK;
    const int fresh = !p.settled || base < 0 ? 0 : base / C8_BLOCK;         // the first chunk that a kernel not yet waited for may have changed
    const size_t to_values = (size_t)p.nkv * per_head * CHUNK;
    bool waited = false;
    int where = 0, scales_next = 0, scales = 0;
    auto look_up = [&](int from) {                                          // chunks begin + from ..
        const int last = min(end, begin + from + 32) - 1;
        const int key = min(begin + from + lane, last) * C8_BLOCK;
        int page = bt[key / p.page_size];
        if (page < 0 || page >= p.num_pages) {
            if (p.status) atomicExch(p.status, 4);
            page = 0;
        }
        where = (page * 2 * p.nkv + g) * per_head + key % p.page_size / C8_BLOCK;
        if (!waited && last >= fresh) {
            // (what the ring takes first is on its way to L2 meanwhile)
            if (lane < min(nt, 2 * D8_STAGES)) {
                d8_prefetch(p.codes + (size_t)where * CHUNK, CHUNK);
                d8_prefetch(p.codes + (size_t)where * CHUNK + to_values, CHUNK);
            }
            pdl_wait();
            waited = true;
        }
        scales_next = c8_scales(p, where, per_head);
    };
    auto bring = [&](int it, int stage) {                                   // chunks begin + 2 it and the next into a place of the ring: K, K, V, V
        if ((it & 15) == 0) look_up(2 * it);
        const int at = __shfl_sync(0xffffffffu, where, (2 * it + (lane & 1)) & 31);
        const bool both = 2 * it + 1 < nt;
        if (lane == 0) mbar_expect_tx(bar + 8 * stage, (both ? 4 : 2) * CHUNK);
        __syncwarp();
        if (lane < 4 && (both || !(lane & 1)))
            d8_copy(ring + (stage * 4 + lane) * CHUNK, p.codes + (size_t)at * CHUNK + (lane & 2 ? to_values : 0), CHUNK, bar + 8 * stage);
    };
    for (int it = 0; it < min(pairs, D8_STAGES); ++it) bring(it, it);
    scales = scales_next;
    if (!waited) { pdl_wait(); waited = true; }                             // q comes from the kernel before this one

    // Q^T: a lane has row gq (and gq + 8), elements 16 tq .. + 15 of each 64; what it needs of the rows of its scores, 2 tq and
    // 2 tq + 1 (and those + 8), comes from the lanes that have them
    float row_f[H][2];
    int row_pos[H][2];
    unsigned qf[H][KS][2];
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const int rr = r0 + gq + 8 * h;
        const bool ok = rr < rows_total;
        const int tok = ok ? rr / n_rep : 0, head = g * n_rep + (ok ? rr - tok * n_rep : 0);
        const __nv_bfloat16* src = q + (size_t)(q0 + tok) * p.q_row_stride + (size_t)head * HD + tq * 16;
        unsigned raw[Q64][8];
        float big = 0.f;
#pragma unroll
        for (int r = 0; r < Q64; ++r) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint4 v = ok ? *reinterpret_cast<const uint4*>(src + r * 64 + half * 8) : make_uint4(0u, 0u, 0u, 0u);
                raw[r][4 * half] = v.x; raw[r][4 * half + 1] = v.y; raw[r][4 * half + 2] = v.z; raw[r][4 * half + 3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                big = fmaxf(big, fmaxf(fabsf(__uint_as_float(raw[r][i] << 16)), fabsf(__uint_as_float(raw[r][i] & 0xffff0000u))));
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // largest element to [2^14, 2^15); the exponent kept where both factors are ordinary numbers
        const int x = min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 127);
        const float up = c8_power(14 - x), down = c8_power(x - 14) * p.scale_log2e;
        const int pos = ok ? base + tok : -1;                               // -1: sees nothing
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const unsigned w = raw[k / 4][2 * (k & 3) + i];
                qf[h][k][i] = d8_half2(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            row_f[h][i] = __shfl_sync(0xffffffffu, down, 4 * (2 * tq + i));
            row_pos[h][i] = __shfl_sync(0xffffffffu, pos, 4 * (2 * tq + i));
        }
    }

    float m[H][2], big[H][2], l[H][2], o[H][HD / 16][4];                    // of rows 2 tq and 2 tq + 1: m, M and the sum of weights
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int i = 0; i < 2; ++i) { m[h][i] = big[h][i] = -INFINITY; l[h][i] = 0.f; }
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) o[h][t][0] = o[h][t][1] = o[h][t][2] = o[h][t][3] = 0.f;
    }
    bool ok = true;

    // Tokens of a chunk in the order of a product's rows: row r < 8 is token r / 2 + 4 (r & 1), row 8 + r the one 8 further on, so that
    // the pairs of rows that a lane of V^T has (2 tq, 2 tq + 1) are tokens tq and 4 + tq.
    const unsigned k_at = ((gq >> 1) + 4 * (gq & 1)) * HD + tq * 16, v_at = tq * HD + gq * (HD / 8);
    const int token = (gq >> 1) + 4 * (gq & 1);
    // N chunks at once (two, or the last one alone): their products do not wait for one another
    auto work = [&](auto number, unsigned kb, int k0, const int (&e)[2]) {
        constexpr int N = decltype(number)::value;
        const unsigned vb = kb + 2 * CHUNK;
        float sc[N][H][4], ev[N];
        bool raise = false;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int h = 0; h < H; ++h) sc[j][h][0] = sc[j][h][1] = sc[j][h][2] = sc[j][h][3] = 0.f;
#pragma unroll
        for (int r = 0; r < Q64; ++r)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint4 ca = d8_lds16(kb + j * CHUNK + k_at + r * 64), cb = d8_lds16(kb + j * CHUNK + k_at + 8 * HD + r * 64);
                const unsigned wa[4] = {ca.x, ca.y, ca.z, ca.w}, wb[4] = {cb.x, cb.y, cb.z, cb.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    unsigned a0, a1, a2, a3;
                    c8_halves4(wa[i], a0, a2);
                    c8_halves4(wb[i], a1, a3);
#pragma unroll
                    for (int h = 0; h < H; ++h) mma_f16_16816(sc[j][h], a0, a1, a2, a3, qf[h][4 * r + i][0], qf[h][4 * r + i][1]);
                }
            }
        const bool edge = k0 + N * C8_BLOCK - 1 > p_min || (p.window > 0 && k0 <= p_max - p.window);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float ek = c8_power((int)(signed char)(e[j] & 0xff));
            ev[j] = (float)(signed char)(e[j] >> 8 & 0xff);
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {                               // row 2 tq + i: its scores of tokens `token` and 8 further on
                    float &x = sc[j][h][i], &y = sc[j][h][2 + i];
                    const float f = row_f[h][i] * ek;
                    x *= f;
                    y *= f;
                    if (edge) {
                        const int pos = row_pos[h][i], kx = k0 + j * C8_BLOCK + token, ky = kx + 8;
                        x = kx <= pos && kx < klen && (p.window <= 0 || kx > pos - p.window) ? x : -INFINITY;
                        y = ky <= pos && ky < klen && (p.window <= 0 || ky > pos - p.window) ? y : -INFINITY;
                    }
                    const float mx = fmaxf(x, y);
                    raise |= mx > m[h][i] + D8_RAISE || mx + ev[j] > big[h][i] + D8_RAISE;
                }
        }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float mx = -INFINITY, rx = -INFINITY;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float x = fmaxf(sc[j][h][i], sc[j][h][2 + i]);
                        mx = fmaxf(mx, x);
                        rx = fmaxf(rx, x + ev[j]);
                    }
#pragma unroll
                    for (int k = 4; k < 32; k *= 2) {
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
                        rx = fmaxf(rx, __shfl_xor_sync(0xffffffffu, rx, k));
                    }
                    if (mx > m[h][i]) {                                     // (m = -inf: the factor is 0, and the sum is 0)
                        l[h][i] *= d8_ex2(m[h][i] - mx);
                        m[h][i] = mx;
                    }
                    if (rx > big[h][i]) {
                        const float f = d8_ex2(big[h][i] - rx);
#pragma unroll
                        for (int t = 0; t < HD / 16; ++t) { o[h][t][i] *= f; o[h][t][2 + i] *= f; }
                        big[h][i] = rx;
                    }
                }
        }
        unsigned pt[N][H][2];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            // (a row that has seen nothing: its scores are -inf, and stay so)
            const float mu[2] = {m[h][0] == -INFINITY ? 0.f : m[h][0], m[h][1] == -INFINITY ? 0.f : m[h][1]};
            const float ru[2] = {m[h][0] == -INFINITY ? 0.f : big[h][0], m[h][1] == -INFINITY ? 0.f : big[h][1]};
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float up = ev[j] - ru[i];
                    w[i] = d8_ex2(sc[j][h][i] + up);
                    w[2 + i] = d8_ex2(sc[j][h][2 + i] + up);
                    l[h][i] += d8_ex2(sc[j][h][i] - mu[i]) + d8_ex2(sc[j][h][2 + i] - mu[i]);
                }
                pt[j][h][0] = d8_turned(d8_half2(w[0], w[1]));
                pt[j][h][1] = d8_turned(d8_half2(w[2], w[3]));
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            // the values of tokens tq, 4 + tq, 8 + tq, 12 + tq: HD / 8 elements from gq * (HD / 8) on
            unsigned v[4][VW];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned at = vb + j * CHUNK + v_at + 4 * i * HD;
                if (HD == 64) {
                    const uint2 x = d8_lds8(at);
                    v[i][0] = x.x; v[i][1] = x.y;
                } else {
                    const uint4 x = d8_lds16(at);
                    v[i][0] = x.x; v[i][1] = x.y; v[i][VW - 2] = x.z; v[i][VW - 1] = x.w;
                }
                const int key = k0 + j * C8_BLOCK + 4 * i + tq;
                if (edge && (key > p_max || key < key_lo)) {                // (what no row sees may be anything)
#pragma unroll
                    for (int c = 0; c < VW; ++c) v[i][c] = 0u;
                }
            }
            // tile t of O^T: rows gq and 8 + gq are elements gq * (HD / 8) + 2t and + 1
#pragma unroll
            for (int c = 0; c < VW; ++c) {
                const unsigned x01[2] = {__byte_perm(v[0][c], v[1][c], 0x5140), __byte_perm(v[0][c], v[1][c], 0x7362)};
                const unsigned x23[2] = {__byte_perm(v[2][c], v[3][c], 0x5140), __byte_perm(v[2][c], v[3][c], 0x7362)};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    unsigned a0, a1, a2, a3;
                    c8_halves4(x01[i], a0, a1);
                    c8_halves4(x23[i], a2, a3);
#pragma unroll
                    for (int h = 0; h < H; ++h) mma_f16_16816(o[h][2 * c + i], a0, a1, a2, a3, pt[j][h][0], pt[j][h][1]);
                }
            }
        }
    };
    int stage = 0, parity = 0;
    for (int it = 0; it < pairs; ++it) {
        if (!__all_sync(0xffffffffu, mbar_wait(bar + 8 * stage, parity))) {
            // given up: the copies that are still under way get one more bounded wait each, then the block leaves
            for (int j = it; j < min(pairs, it + D8_STAGES); ++j) mbar_wait(bar + 8 * (j % D8_STAGES), (j / D8_STAGES) & 1);
            ok = false;
            break;
        }
        const unsigned kb = ring + stage * 4 * CHUNK;
        const int k0 = (begin + 2 * it) * C8_BLOCK;
        const int e[2] = {__shfl_sync(0xffffffffu, scales, (2 * it) & 31), __shfl_sync(0xffffffffu, scales, (2 * it + 1) & 31)};
        if (2 * it + 1 < nt) work(Number<2>(), kb, k0, e);
        else work(Number<1>(), kb, k0, e);
        __syncwarp();                                                       // every lane has what it wants of this place
        if (it + D8_STAGES < pairs) bring(it + D8_STAGES, stage);
        if ((it & 15) == 15) scales = scales_next;                          // (the look-up of the next 32 is behind us)
        if (++stage == D8_STAGES) { stage = 0; parity ^= 1; }
    }
    if (!ok) failed = 1;
    __syncwarp();

    // ---- the warps' results, joined in warp order; a warp's own part of the ring holds its O (all its copies have arrived)
    float* wO = reinterpret_cast<float*>(d8_smem + (size_t)warp * D8_WARP_BYTES<HD>);
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = 8 * h + 2 * tq + i;
            float sum = l[h][i];
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            if (gq == 0) { sM[warp][row] = m[h][i]; sR[warp][row] = big[h][i]; sL[warp][row] = sum; }
#pragma unroll
            for (int t = 0; t < HD / 16; t += 2)
                *reinterpret_cast<float4*>(wO + row * HD + gq * (HD / 8) + 2 * t) =
                    make_float4(o[h][t][i], o[h][t][2 + i], o[h][t + 1][i], o[h][t + 1][2 + i]);
        }
    __syncthreads();
    // a row's result is (O / l) 2^(M - m), the power in two halves so that neither leaves float's range
    auto store = [&](int r, int c, float4 x, float sum, float up) {
        const int rr = r0 + r;
        if (rr >= rows_total || failed) return;
        const int tok = rr / n_rep, head = g * n_rep + rr - tok * n_rep;
        const float inv = sum == 0.f ? 0.f : 1.f / sum, f = sum == 0.f ? 0.f : d8_ex2(0.5f * up);        // a row that sees nothing: zeros
        const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x * inv * f * f, x.y * inv * f * f), hi = __floats2bfloat162_rn(x.z * inv * f * f, x.w * inv * f * f);
        *reinterpret_cast<uint2*>(out + ((size_t)(q0 + tok) * p.nh + head) * HD + c) =
            make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
    };
    for (int i = threadIdx.x; i < ROWS * HD / 4; i += WARPS * 32) {
        const int r = i / (HD / 4), c = i % (HD / 4) * 4;
        float mx = -INFINITY, rx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) { mx = fmaxf(mx, sM[w][r]); rx = fmaxf(rx, sR[w][r]); }
        const float mu = mx == -INFINITY ? 0.f : mx, ru = rx == -INFINITY ? 0.f : rx;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float a = d8_ex2(sR[w][r] - ru);
            const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(d8_smem + (size_t)w * D8_WARP_BYTES<HD>) + r * HD + c);
            sum = fmaf(sL[w][r], d8_ex2(sM[w][r] - mu), sum);
            x.x = fmaf(y.x, a, x.x); x.y = fmaf(y.y, a, x.y); x.z = fmaf(y.z, a, x.z); x.w = fmaf(y.w, a, x.w);
        }
        if (splits == 1) {
            store(r, c, x, sum, ru - mu);
        } else {
            *reinterpret_cast<float4*>(&xO[r][c]) = x;
            if (c == 0) { xM[r] = mx; xR[r] = rx; xL[r] = sum; }
        }
    }
    if (splits > 1) {
        cluster_sync();                                                     // every block's result is in place
        // (each block pieces that follow one another: neighbours' reads of another block's memory are then one)
        const int mine = (ROWS * HD / 4 + splits - 1) / splits;
        for (int i = rank * mine + threadIdx.x; i < min((rank + 1) * mine, ROWS * HD / 4); i += WARPS * 32) {
            const int r = i / (HD / 4), c = i % (HD / 4) * 4;
            float mx = -INFINITY, rx = -INFINITY, sum = 0.f;
            for (int j = 0; j < splits; ++j) {
                mx = fmaxf(mx, cluster_f32(cluster_peer(&xM[r], (unsigned)j)));
                rx = fmaxf(rx, cluster_f32(cluster_peer(&xR[r], (unsigned)j)));
            }
            const float mu = mx == -INFINITY ? 0.f : mx, ru = rx == -INFINITY ? 0.f : rx;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int j = 0; j < splits; ++j) {
                const float a = d8_ex2(cluster_f32(cluster_peer(&xR[r], (unsigned)j)) - ru), b = d8_ex2(cluster_f32(cluster_peer(&xM[r], (unsigned)j)) - mu);
                const float4 y = cluster_f32x4(cluster_peer(&xO[r][c], (unsigned)j));
                sum = fmaf(cluster_f32(cluster_peer(&xL[r], (unsigned)j)), b, sum);
                x.x = fmaf(y.x, a, x.x); x.y = fmaf(y.y, a, x.y); x.z = fmaf(y.z, a, x.z); x.w = fmaf(y.w, a, x.w);
            }
            store(r, c, x, sum, ru - mu);
        }
        cluster_sync();                                                     // nobody reads this block's memory any more
    }
    if (threadIdx.x == 0 && failed && p.status) atomicExch(p.status, 16);
}

// The limits that a device has to allow, asked once per device: shared memory, clusters of more than 8 blocks.
template <int HD, bool WIDE, int WARPS>
static int decode8_ready() {
    static int done[64] = {0};                     // 0 unknown, 1 yes
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(-101, "paged_attention8: cannot tell the current device");
    if (!done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(decode8_kernel<HD, WIDE, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)D8_SMEM<HD, WARPS>);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(decode8_kernel<HD, WIDE, WARPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return fail(-101, "paged_attention8: cannot reserve %zu bytes of shared memory: %s", D8_SMEM<HD, WARPS>, cudaGetErrorString(e));
        done[dev] = 1;
    }
    return 0;
}
// blocks of the kernel that the device holds at a time
template <int HD>
static int decode8_slots() {
    static int per_sm = 0;                         // (the same on every device that the kernel is built for)
    if (per_sm == 0 && (decode8_ready<HD, false, D8_WARPS>() != 0 ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, decode8_kernel<HD, false, D8_WARPS>, D8_WARPS * 32, D8_SMEM<HD, D8_WARPS>) != cudaSuccess || per_sm <= 0)) {
        cudaGetLastError();
        per_sm = 0;
        return 2 * sm_count();
    }
    return sm_count() * per_sm;
}

template <int HD, bool WIDE, int WARPS>
static int launch_decode8_of(const C8Params& p, const void* q, void* out, int num_seqs, long long rows, int splits, int most_q, cudaStream_t stream) {
    const int rc = decode8_ready<HD, WIDE, WARPS>();
    if (rc != 0) return rc;
    const long long tiles = (rows + (WIDE ? 15 : 7)) / (WIDE ? 16 : 8);
    if (tiles * splits > 0x7fffffffLL || p.nkv > 65535 || num_seqs > 65535)
        return fail(-1, "paged_attention8: the step exceeds the grid (%lld row tiles, %d kv heads, %d sequences)", tiles, p.nkv, num_seqs);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * splits), p.nkv, num_seqs);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = D8_SMEM<HD, WARPS>;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return check_launch("paged_attention8", cudaLaunchKernelEx(&cfg, decode8_kernel<HD, WIDE, WARPS>, p, (const __nv_bfloat16*)q, (__nv_bfloat16*)out, splits, most_q));
}

// sequences that bring more than `most_q` tokens are left alone
template <int HD>
static int launch_decode8(const C8Params& p, const void* q, void* out, int num_seqs, int max_q, int max_k, int splits, int most_q, cudaStream_t stream) {
    if (splits < 1) splits = 1;
    if (splits > D8_MAX_CLUSTER) return fail(-1, "paged_attention8: %d splits are more than %d", splits, D8_MAX_CLUSTER);
    const long long rows = (long long)(max_q < most_q ? max_q : most_q) * (p.nh / p.nkv);
    // Blocks of four warps where not all of eight would be on the device at once and a sequence's keys (or the window's) are few: a block's time is then
    // mostly its start, its first copies' way and its join, and twice as many are under way.  us with eight and with four, 32 / 8 heads of 64: 64 requests of
    // 64 keys 7.9 / 4.4, 300 10.2 / 6.7, 60 to 500 10.3 / 7.9, 125 to 1,000 13.7 / 12.5; 40 of 1,000 14.4 / 14.0; but 64 of 128 to 2,048 19.8 / 22.0, whose longest
    // are then alone for longer, and 64 of 60 to 500 with half the heads, all at once, 5.4 / 6.8.
    const long long blocks = (rows + (rows <= 8 ? 7 : 15)) / (rows <= 8 ? 8 : 16) * p.nkv * num_seqs;
    const bool few = splits == 1 && blocks > decode8_slots<HD>() && (max_k <= 1024 || (p.window > 0 && p.window <= 1024));
    if (rows <= 8) return few ? launch_decode8_of<HD, false, D8_FEW_WARPS>(p, q, out, num_seqs, rows, splits, most_q, stream)
                              : launch_decode8_of<HD, false, D8_WARPS>(p, q, out, num_seqs, rows, splits, most_q, stream);
    return few ? launch_decode8_of<HD, true, D8_FEW_WARPS>(p, q, out, num_seqs, rows, splits, most_q, stream)
               : launch_decode8_of<HD, true, D8_WARPS>(p, q, out, num_seqs, rows, splits, most_q, stream);
}

}  // namespace vapi
