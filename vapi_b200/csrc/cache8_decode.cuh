// Attention over an 8-bit cache on the tensor cores (mma.sync m16n8k16, f16 in, float accumulate): bfloat16 queries, head size 64
// or 128, any page size and any number of rows.
//
// A decode step reads every key and value of every live request once, so the kernel is built around that stream.  A cluster of
// up to 16 blocks owns one (sequence, kv head, tile of 8 or 16 rows) and its eight warps each a run of chunks: the 16
// tokens that share a scale, one piece of memory of 16 * head size bytes for K and one for V.  A warp brings its own chunks
// in by bulk copies through a ring of its own, and no warp waits for another before the end, where their partial results are
// joined: through shared memory in a block, through the cluster's among its blocks, always in the same order.
//
//   S = Q K^T    A code is an f16 number exactly.  A row of Q is scaled by a power of two so that its largest element is near
//                2^14: f16 then has three bits more than bfloat16 for it, and elements keep all of theirs down to 2^-28 of the
//                largest.  A lane's 16 contiguous bytes of a key are its B operands of four k-steps: the order of the head's
//                elements in the sum is free as long as Q follows it, and so no byte moves between lanes.
//   O += P V     P = 2^(s - m_chunk) with the chunk's own row maximum, so that its largest is 1 whatever the other chunks hold;
//                the chunk's product is added to O times 2^(m_chunk - m + e_V) in float.  (P times the scale in f16 would lose
//                what a block of small values says beside one of large.)  The values of two tokens are paired by byte
//                permutes; which token is which k is free too, as long as K's columns follow.
//
// Keys behind a sequence's end are masked by selection, and their values taken as zeros.  (A NaN among the keys and values that a
// sequence did write, though a row may not see it, can reach that row through 0 * NaN; the step that wrote it was lost.)
#pragma once
#include "cache8.cuh"
#include "cluster.cuh"
#include "tcgen05.cuh"           // mbarriers with bounded waits

namespace vapi {

constexpr int D8_WARPS = 8;
constexpr int D8_MAX_CLUSTER = 16;
template <int HD> constexpr int D8_STAGES = HD == 64 ? 6 : 3;
template <int HD> constexpr int D8_CHUNK = C8_BLOCK * HD;                              // bytes of a chunk of K, or of V
template <int HD> constexpr int D8_WARP_BYTES = D8_STAGES<HD> * 2 * D8_CHUNK<HD>;
template <int HD> constexpr size_t D8_SMEM = (size_t)D8_WARPS * D8_WARP_BYTES<HD>;

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
// WIDE: tiles of 16 rows; else of 8 (the lower half of every fragment is then zero and is not worked out).
template <int HD, bool WIDE>
__global__ void __launch_bounds__(D8_WARPS * 32, 2)
decode8_kernel(const C8Params p, const __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ out, const int splits, const int most_q) {
    constexpr int ROWS = WIDE ? 16 : 8, H = WIDE ? 2 : 1, STAGES = D8_STAGES<HD>, CHUNK = D8_CHUNK<HD>;
    constexpr int KS = HD / 16, NT = HD / 8, Q64 = HD / 64;                 // k-steps of S, column tiles of O, runs of 64 elements
    extern __shared__ __align__(128) unsigned char d8_smem[];
    __shared__ __align__(8) unsigned long long bars[D8_WARPS * STAGES];
    __shared__ float sM[D8_WARPS][ROWS], sL[D8_WARPS][ROWS];
    __shared__ float xM[ROWS], xL[ROWS];
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
    const int units = splits * D8_WARPS, unit = rank * D8_WARPS + warp;
    const int begin = c_lo + (int)(chunks * unit / units), end = c_lo + (int)(chunks * (unit + 1) / units), nt = end - begin;

    const unsigned bar = smem_u32(bars + warp * STAGES), ring = smem_u32(d8_smem + (size_t)warp * D8_WARP_BYTES<HD>);
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(bar + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 0) failed = 0;
    __syncthreads();

    // Where 32 chunks at a time lie, one a lane, and their scales: looked up as the copies reach them, used as the products do.
    const int* bt = p.block_table + (size_t)s * p.table_stride;
    const int per_head = p.page_size / C8_BLOCK;
    const int fresh = base < 0 ? 0 : base / C8_BLOCK;                       // the first chunk that this step's tokens may have changed
    bool waited = false;
    int where = 0, scales_next = 0, scales = 0;
    auto look_up = [&](int from) {                                          // chunks begin + from ..
        const int last = min(end, begin + from + 32) - 1;
        if (!waited && last >= fresh) { pdl_wait(); waited = true; }
        const int key = min(begin + from + lane, last) * C8_BLOCK;
        int page = bt[key / p.page_size];
        if (page < 0 || page >= p.num_pages) {
            if (p.status) atomicExch(p.status, 4);
            page = 0;
        }
        where = (page * 2 * p.nkv + g) * per_head + key % p.page_size / C8_BLOCK;
        scales_next = c8_scales(p, where, per_head);
    };
    auto bring = [&](int it) {                                              // chunk begin + it into its place of the ring
        if ((it & 31) == 0) look_up(it);
        const int at = __shfl_sync(0xffffffffu, where, it & 31), stage = it % STAGES;
        if (lane == 0) {
            mbar_expect_tx(bar + 8 * stage, 2 * CHUNK);
            const unsigned dst = ring + stage * 2 * CHUNK;
            d8_copy(dst, p.codes + (size_t)at * CHUNK, CHUNK, bar + 8 * stage);
            d8_copy(dst + CHUNK, p.codes + ((size_t)at + (size_t)p.nkv * per_head) * CHUNK, CHUNK, bar + 8 * stage);
        }
    };
    for (int it = 0; it < min(nt, STAGES); ++it) bring(it);
    scales = scales_next;
    if (!waited) { pdl_wait(); waited = true; }                             // q comes from the kernel before this one

    int row_pos[H];
    float row_f[H];
    unsigned qf[KS][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (h >= H) {
#pragma unroll
            for (int k = 0; k < KS; ++k) qf[k][1] = qf[k][3] = 0u;
            break;
        }
        const int rr = r0 + gq + 8 * h;
        const bool ok = rr < rows_total;
        const int tok = ok ? rr / n_rep : 0, head = g * n_rep + (ok ? rr - tok * n_rep : 0);
        row_pos[h] = ok ? base + tok : -1;                                  // -1: sees nothing
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
        const int x = min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 120);
        const float up = c8_power(14 - x);
        row_f[h] = c8_power(x - 14) * p.scale_log2e;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const unsigned a = raw[k / 4][2 * (k & 3)], b = raw[k / 4][2 * (k & 3) + 1];
            qf[k][h] = d8_half2(__uint_as_float(a << 16) * up, __uint_as_float(a & 0xffff0000u) * up);
            qf[k][2 + h] = d8_half2(__uint_as_float(b << 16) * up, __uint_as_float(b & 0xffff0000u) * up);
        }
    }

    float m[H], l[H], o[NT][2 * H];
#pragma unroll
    for (int h = 0; h < H; ++h) { m[h] = -INFINITY; l[h] = 0.f; }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2 * H; ++i) o[t][i] = 0.f;
    bool ok = true;

    for (int it = 0; it < nt; ++it) {
        const int stage = it % STAGES, k0 = (begin + it) * C8_BLOCK;
        if (!__all_sync(0xffffffffu, mbar_wait(bar + 8 * stage, (it / STAGES) & 1))) {
            // given up: the copies that are still under way get one more bounded wait each, then the block leaves
            for (int j = it; j < min(nt, it + STAGES); ++j) mbar_wait(bar + 8 * (j % STAGES), (j / STAGES) & 1);
            ok = false;
            break;
        }
        const unsigned kb = ring + stage * 2 * CHUNK, vb = kb + CHUNK;
        // scores of tokens 8j + (column / 2) + 4 (column & 1), in tile j
        float sc[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
            const unsigned row = kb + (8 * j + (gq >> 1) + 4 * (gq & 1)) * HD + tq * 16;
#pragma unroll
            for (int r = 0; r < Q64; ++r) {
                const uint4 c = d8_lds16(row + r * 64);
                const unsigned w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mma_f16_16816(sc[j], qf[4 * r + i][0], qf[4 * r + i][1], qf[4 * r + i][2], qf[4 * r + i][3],
                                  c8_halves((unsigned short)(w[i] & 0xffffu)), c8_halves((unsigned short)(w[i] >> 16)));
            }
        }
        // the values of tokens tq, 4 + tq, 8 + tq, 12 + tq: HD / 8 elements from gq * (HD / 8) on
        unsigned v[4][NT / 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned at = vb + (4 * i + tq) * HD + gq * (HD / 8);
            if (HD == 64) {
                const uint2 x = d8_lds8(at);
                v[i][0] = x.x; v[i][1] = x.y;
            } else {
                const uint4 x = d8_lds16(at);
                v[i][0] = x.x; v[i][1] = x.y; v[i][NT / 4 - 2] = x.z; v[i][NT / 4 - 1] = x.w;
            }
            if (k0 + C8_BLOCK > klen && k0 + 4 * i + tq >= klen) {
#pragma unroll
                for (int c = 0; c < NT / 4; ++c) v[i][c] = 0u;
            }
        }
        const int e = __shfl_sync(0xffffffffu, scales, it & 31);
        __syncwarp();                                                       // every lane has what it wants of this place
        if (it + STAGES < nt) bring(it + STAGES);
        if ((it & 31) == 31) scales = scales_next;                          // (the look-up of the next 32 is behind us: STAGES < 32)

        const float ek = c8_power((int)(signed char)(e & 0xff)), ev = c8_power((int)(signed char)(e >> 8 & 0xff));
        const bool edge = k0 + C8_BLOCK - 1 > p_min || (p.window > 0 && k0 <= p_max - p.window);
        float add[H];
        bool moved = false;
        float keep[H];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const float f = row_f[h] * ek;
            float* x[4] = {&sc[0][2 * h], &sc[0][2 * h + 1], &sc[1][2 * h], &sc[1][2 * h + 1]};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *x[i] *= f;
                if (edge) {
                    const int key = k0 + 4 * i + tq;                        // column 2 tq + (i & 1) of tile i >> 1
                    const bool sees = key <= row_pos[h] && key < klen && (p.window <= 0 || key > row_pos[h] - p.window);
                    *x[i] = sees ? *x[i] : -INFINITY;
                }
            }
            float mx = fmaxf(fmaxf(*x[0], *x[1]), fmaxf(*x[2], *x[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mu = mx == -INFINITY ? 0.f : mx, mn = fmaxf(m[h], mx), mnu = mn == -INFINITY ? 0.f : mn;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *x[i] = d8_ex2(*x[i] - mu);
                sum += *x[i];
            }
            const float a = d8_ex2(m[h] - mnu), b = d8_ex2(mx - mnu);
            l[h] = l[h] * a + sum * b;
            m[h] = mn;
            keep[h] = a;
            add[h] = b * ev;
            moved |= a != 1.f;
        }
        const unsigned a0 = d8_half2(sc[0][0], sc[0][1]), a2 = d8_half2(sc[1][0], sc[1][1]);
        const unsigned a1 = WIDE ? d8_half2(sc[0][2], sc[0][3]) : 0u, a3 = WIDE ? d8_half2(sc[1][2], sc[1][3]) : 0u;
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 2 * H; ++i) o[t][i] *= keep[i >> 1];
        }
#pragma unroll
        for (int c = 0; c < NT / 4; ++c) {
            const unsigned lo01 = __byte_perm(v[0][c], v[1][c], 0x5140), hi01 = __byte_perm(v[0][c], v[1][c], 0x7362);
            const unsigned lo23 = __byte_perm(v[2][c], v[3][c], 0x5140), hi23 = __byte_perm(v[2][c], v[3][c], 0x7362);
            const unsigned w01[2] = {lo01, hi01}, w23[2] = {lo23, hi23};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned x = w01[i >> 1], y = w23[i >> 1];
                float t4[4] = {0.f, 0.f, 0.f, 0.f};
                mma_f16_16816(t4, a0, a1, a2, a3, c8_halves((unsigned short)(i & 1 ? x >> 16 : x & 0xffffu)),
                              c8_halves((unsigned short)(i & 1 ? y >> 16 : y & 0xffffu)));
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    o[4 * c + i][2 * h] = fmaf(t4[2 * h], add[h], o[4 * c + i][2 * h]);
                    o[4 * c + i][2 * h + 1] = fmaf(t4[2 * h + 1], add[h], o[4 * c + i][2 * h + 1]);
                }
            }
        }
    }
    if (!ok) failed = 1;
    __syncwarp();

    // ---- the warps' results, joined in warp order; a warp's own part of the ring holds its O (all its copies have arrived)
    float* wO = reinterpret_cast<float*>(d8_smem + (size_t)warp * D8_WARP_BYTES<HD>);
#pragma unroll
    for (int h = 0; h < H; ++h) {
        float sum = l[h];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (tq == 0) { sM[warp][gq + 8 * h] = m[h]; sL[warp][gq + 8 * h] = sum; }
        // columns 2 tq and 2 tq + 1 of tile t are elements (2 tq) * NT + t and (2 tq + 1) * NT + t
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < NT; t += 4)
                *reinterpret_cast<float4*>(wO + (gq + 8 * h) * HD + (2 * tq + i) * NT + t) =
                    make_float4(o[t][2 * h + i], o[t + 1][2 * h + i], o[t + 2][2 * h + i], o[t + 3][2 * h + i]);
    }
    __syncthreads();
    auto store = [&](int r, int c, float4 x, float sum) {
        const int rr = r0 + r;
        if (rr >= rows_total || failed) return;
        const int tok = rr / n_rep, head = g * n_rep + rr - tok * n_rep;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;                     // a row that sees nothing: zeros
        const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x * inv, x.y * inv), hi = __floats2bfloat162_rn(x.z * inv, x.w * inv);
        *reinterpret_cast<uint2*>(out + ((size_t)(q0 + tok) * p.nh + head) * HD + c) =
            make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
    };
    for (int i = threadIdx.x; i < ROWS * HD / 4; i += D8_WARPS * 32) {
        const int r = i / (HD / 4), c = i % (HD / 4) * 4;
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < D8_WARPS; ++w) mx = fmaxf(mx, sM[w][r]);
        const float mu = mx == -INFINITY ? 0.f : mx;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < D8_WARPS; ++w) {
            const float a = d8_ex2(sM[w][r] - mu);
            const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(d8_smem + (size_t)w * D8_WARP_BYTES<HD>) + r * HD + c);
            sum = fmaf(sL[w][r], a, sum);
            x.x = fmaf(y.x, a, x.x); x.y = fmaf(y.y, a, x.y); x.z = fmaf(y.z, a, x.z); x.w = fmaf(y.w, a, x.w);
        }
        if (splits == 1) {
            store(r, c, x, sum);
        } else {
            *reinterpret_cast<float4*>(&xO[r][c]) = x;
            if (c == 0) { xM[r] = mx; xL[r] = sum; }
        }
    }
    if (splits > 1) {
        cluster_sync();                                                  // every block's result is in place
        for (int i = threadIdx.x * splits + rank; i < ROWS * HD / 4; i += D8_WARPS * 32 * splits) {
            const int r = i / (HD / 4), c = i % (HD / 4) * 4;
            float mx = -INFINITY, sum = 0.f;
            for (int j = 0; j < splits; ++j) mx = fmaxf(mx, cluster_f32(cluster_peer(&xM[r], (unsigned)j)));
            const float mu = mx == -INFINITY ? 0.f : mx;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int j = 0; j < splits; ++j) {
                const float a = d8_ex2(cluster_f32(cluster_peer(&xM[r], (unsigned)j)) - mu);
                const float4 y = cluster_f32x4(cluster_peer(&xO[r][c], (unsigned)j));
                sum = fmaf(cluster_f32(cluster_peer(&xL[r], (unsigned)j)), a, sum);
                x.x = fmaf(y.x, a, x.x); x.y = fmaf(y.y, a, x.y); x.z = fmaf(y.z, a, x.z); x.w = fmaf(y.w, a, x.w);
            }
            store(r, c, x, sum);
        }
        cluster_sync();                                                  // nobody reads this block's memory any more
    }
    if (threadIdx.x == 0 && failed && p.status) atomicExch(p.status, 16);
}

// The limits that a device has to allow, asked once per device: shared memory, clusters of more than 8 blocks.
template <int HD, bool WIDE>
static int decode8_ready() {
    static int done[64] = {0};                     // 0 unknown, 1 yes
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(-101, "paged_attention8: cannot tell the current device");
    if (!done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(decode8_kernel<HD, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)D8_SMEM<HD>);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(decode8_kernel<HD, WIDE>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return fail(-101, "paged_attention8: cannot reserve %zu bytes of shared memory: %s", D8_SMEM<HD>, cudaGetErrorString(e));
        done[dev] = 1;
    }
    return 0;
}
// blocks of the kernel that the device holds at a time
template <int HD>
static int decode8_slots() {
    static int per_sm = 0;                         // (the same on every device that the kernel is built for)
    if (per_sm == 0 && (decode8_ready<HD, false>() != 0 ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, decode8_kernel<HD, false>, D8_WARPS * 32, D8_SMEM<HD>) != cudaSuccess || per_sm <= 0)) {
        cudaGetLastError();
        per_sm = 0;
        return 2 * sm_count();
    }
    return sm_count() * per_sm;
}

template <int HD, bool WIDE>
static int launch_decode8_of(const C8Params& p, const void* q, void* out, int num_seqs, long long rows, int splits, int most_q, cudaStream_t stream) {
    const int rc = decode8_ready<HD, WIDE>();
    if (rc != 0) return rc;
    const long long tiles = (rows + (WIDE ? 15 : 7)) / (WIDE ? 16 : 8);
    if (tiles * splits > 0x7fffffffLL || p.nkv > 65535 || num_seqs > 65535)
        return fail(-1, "paged_attention8: the step exceeds the grid (%lld row tiles, %d kv heads, %d sequences)", tiles, p.nkv, num_seqs);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * splits), p.nkv, num_seqs);
    cfg.blockDim = dim3(D8_WARPS * 32);
    cfg.dynamicSmemBytes = D8_SMEM<HD>;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return check_launch("paged_attention8", cudaLaunchKernelEx(&cfg, decode8_kernel<HD, WIDE>, p, (const __nv_bfloat16*)q, (__nv_bfloat16*)out, splits, most_q));
}

template <int HD>
// sequences that bring more than `most_q` tokens are left alone
static int launch_decode8(const C8Params& p, const void* q, void* out, int num_seqs, int max_q, int splits, int most_q, cudaStream_t stream) {
    if (splits < 1) splits = 1;
    if (splits > D8_MAX_CLUSTER) return fail(-1, "paged_attention8: %d splits are more than %d", splits, D8_MAX_CLUSTER);
    const long long rows = (long long)(max_q < most_q ? max_q : most_q) * (p.nh / p.nkv);
    if (rows <= 8) return launch_decode8_of<HD, false>(p, q, out, num_seqs, rows, splits, most_q, stream);
    return launch_decode8_of<HD, true>(p, q, out, num_seqs, rows, splits, most_q, stream);
}

}  // namespace vapi
