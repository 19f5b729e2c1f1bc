// Products of a 4-bit weight with more rows than int4_rows_kernel takes, on the fifth-generation tensor cores (tcgen05): the codes become bfloat16
// numbers, (code - zero) * scale rounded once, on their way to shared memory, and never stand in memory as such.
//
// A block owns 128 features (for a gated product 64 of the gate and the same 64 of up) and N rows of x; the blocks of a cluster share out the
// columns.  A chunk is 64 columns:
//   warps 0..7  a tile row of codes each (int4.cu says how it lies), AHEAD chunks under way in registers; what they make of it goes to a ring of
//               stages in tensor memory, where a product may have its first operand: the codes' order is that of a 16-lane store.  (Through
//               shared memory W was written there and read again, 32 of a chunk's 56 KB at 64 rows, and that was what bounded the kernel.)
//   warp 8      x, by TMA into a ring of shared-memory stages (rows and columns behind the end are zeros);
//   warp 9      D[feature][row] += W X^T, issued by one lane of the whole warp; owns the tensor memory.
// Then warps 0..7 bring D to shared memory, where x's stages were, and all threads write what comes of it, four features at a time.
//
// What bounds it: making the numbers.  A chunk is 64 conversions a lane of eight warps beside barriers and the store, 430 cycles of a warp one after
// the other, and about as many of a multiprocessor with two blocks on it; the products of 64 rows take 180, the bytes of a chunk's codes 190.  64
// rows of 8,192 x 28,672 in 45 us (2.7 TB/s of codes; with 16-bit weights the product takes 76), of 16,384 x 2,048 gated in 11.0 (9.6), of 2,048 x
// 8,192 in 11.4 (11.9); 2,048 rows of 2,048 x 8,192 in 48 us, 1.43 PFLOP/s, and in 61 where one pass follows another (the power cap).
//
// Every wait is bounded; a role that gives up marks the block, whose sums are then NaN, and so is every result of its cluster, which adds them up.  The
// products and copies that are under way are awaited first.
#pragma once
#include "cluster.cuh"
#include "tcgen05.cuh"

namespace vapi {

constexpr int I4T_LOADERS = 8, I4T_THREADS = (I4T_LOADERS + 2) * 32, I4T_FEATURES = 128, I4T_AHEAD = 6;
template <int N> constexpr int I4T_STAGES = N <= 64 ? 6 : 4;
template <int N> constexpr int I4T_BLOCKS = N > 128 ? 1 : 2;                                  // a multiprocessor
template <int N> constexpr int I4T_STAGE = N * 128;                                           // bytes of x
template <int N> constexpr int I4T_COLUMNS = N > 128 ? 512 : 256;                             // of tensor memory: D, then 32 a stage of W
template <int N> constexpr size_t I4T_SMEM = 1024 + (size_t)I4T_STAGES<N> * I4T_STAGE<N> + 256;

// D += A B^T with A in tensor memory, a row a lane and two k a column
__device__ __forceinline__ void i4t_mma(unsigned d, unsigned a, unsigned long long b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}

// GS: k-steps of 16 columns a group (2, 4, 8).  TRIAL: the blocks of one rank give up at their first wait (p.trial; for tests)
template <int N, int GS, bool GLU, bool TRIAL>
__global__ void __launch_bounds__(I4T_THREADS, I4T_BLOCKS<N>)
int4_tile_kernel(const __grid_constant__ CUtensorMap tm_x, const I4Params p, const int splits) {
    constexpr int STAGES = I4T_STAGES<N>, STAGE = I4T_STAGE<N>, COLUMNS = I4T_COLUMNS<N>, AHEAD = I4T_AHEAD, GPC = GS < 4 ? 2 : 1, CPG = GS > 4 ? 2 : 1;
    static_assert(N * I4T_FEATURES * 4 <= STAGES * STAGE, "D fits where the stages were");
    static_assert(N + 32 * STAGES <= COLUMNS && COLUMNS * I4T_BLOCKS<N> <= 512, "D and W fit in tensor memory");
    extern __shared__ unsigned char i4t_smem[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(i4t_smem) + 1023) & ~(uintptr_t)1023);
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(base + (size_t)STAGES * STAGE);
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + 3 * STAGES + 2);
    volatile int* failed = reinterpret_cast<int*>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x % splits, block = (int)blockIdx.x / splits, r0 = (int)blockIdx.y * N;
    const int from = (int)((long long)p.chunks * rank / splits), upto = (int)((long long)p.chunks * (rank + 1) / splits);
    const unsigned full = smem_u32(bars), empty = smem_u32(bars + STAGES), x_full = smem_u32(bars + 2 * STAGES), done = smem_u32(bars + 3 * STAGES);
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(full + 8 * i, 8); mbar_init(empty + 8 * i, 1); mbar_init(x_full + 8 * i, 1); }
        mbar_init(done, 1);
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == I4T_LOADERS + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((unsigned)COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    pdl_trigger();                                 // (not before the allocation: a block of the next kernel that came between would be waited for, and wait)
    const unsigned tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const bool give_up = TRIAL && rank == p.trial;

    if (warp < I4T_LOADERS) {
        // (a warp reaches the lanes of one quarter of tensor memory: two tile rows)
        const int g = lane >> 2, tiles = (p.n + 15) / 16, groups = GS < 4 ? 2 * p.chunks : p.k / p.group, tn = 2 * (warp & 3) + (warp >> 2);
        const int mine = GLU ? (tn < 4 ? block * 4 + tn : tiles / 2 + block * 4 + tn - 4) : block * 8 + tn;
        const bool real = GLU ? block * 4 + (tn & 3) < tiles / 2 : mine < tiles;
        const unsigned to_w = tmem + N + ((unsigned)(16 * tn) << 16);
        const uint4* codes = reinterpret_cast<const uint4*>(p.codes) + (size_t)(real ? mine : 0) * p.chunks * 32 + lane;
        const uint2* scales = reinterpret_cast<const uint2*>(p.scales) + (size_t)(real ? mine : 0) * groups * 8 + g;
        uint4 w[AHEAD];
        uint2 sc[AHEAD][GPC];
        auto bring = [&](int ch, uint4& to, uint2 (&ts)[GPC]) {
            if (ch >= upto) return;
            to = __ldg(codes + (size_t)ch * 32);
#pragma unroll
            for (int i = 0; i < GPC; ++i) ts[i] = __ldg(scales + (size_t)(ch / CPG * GPC + i) * 8);
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) bring(from + i, w[i], sc[i]);
        int stage = 0, parity = 1;
        bool ok = true, free = true;               // (the first stages are)
        for (int at = from; at < upto && ok; at += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int ch = at + i;
                if (ch >= upto) break;
                if (!__all_sync(0xffffffffu, free) && (give_up || !mbar_wait_warp(empty + 8 * stage, parity))) { ok = false; break; }
                tc5_fence_after();
                // (the next stage asked for before this one is made: 8,192 x 28,672, 64 rows 45.8 to 44.7 us; small ones the same)
                const int next = stage + 1 == STAGES ? 0 : stage + 1;
                free = mbar_ended(empty + 8 * next, next == 0 ? parity ^ 1 : parity);
                const unsigned words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                unsigned v[16];                    // word 2j + q of a row's 8 words a lane: of row g, of row g + 8
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint2 of = sc[i][GPC == 2 ? j >> 1 : 0];
                        const unsigned pair = h ? of.y : of.x, both = __byte_perm(pair, pair, 0x1010);
                        const __nv_bfloat162 zero = i4_zero(pair), scale = *reinterpret_cast<const __nv_bfloat162*>(&both);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const unsigned u = i4_pair(words[j], 8 * q + 4 * h, zero);
                            const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&u), scale);
                            v[2 * (2 * j + q) + h] = *reinterpret_cast<const unsigned*>(&y);
                        }
                    }
                asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                             ::"r"(to_w + 32 * stage), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                               "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
                tmem_st_wait();
                tc5_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(full + 8 * stage);
                bring(ch + AHEAD, w[i], sc[i]);
                if (next == 0) parity ^= 1;
                stage = next;
            }
        }
        if (ok && upto > from && !mbar_wait_warp(done, 0)) ok = false;
        if (!ok) *failed = 1;
        __syncthreads();
        tc5_fence_after();
        // D to shared memory, [row][feature]: every product has ended, and so nothing reads the stages
        const bool bad = *failed != 0;             // (of any role: all have been here)
        const int quarter = warp & 3, column = (warp >> 2) * (N / 2);
        float* d = reinterpret_cast<float*>(base) + quarter * 32 + lane;
        if (upto > from) {
#pragma unroll 2
            for (int j = 0; j < N / 2; j += 16) {
                float v[16];
                tmem_ld16(tmem + ((unsigned)(quarter * 32) << 16) + column + j, v);
#pragma unroll
                for (int e = 0; e < 16; ++e) d[(column + j + e) * I4T_FEATURES] = bad ? __int_as_float(0x7fc00000) : v[e];
            }
        } else {
            for (int j = 0; j < N / 2; ++j) d[(column + j) * I4T_FEATURES] = 0.f;
        }
    } else if (warp == I4T_LOADERS) {
        if (lane == 0) {
            pdl_wait();                            // x comes from the kernel before this one
            int stage = 0, parity = 1, asked = 0;
            for (int ch = from; ch < upto; ++ch, ++asked) {
                if (give_up || !mbar_wait(empty + 8 * stage, parity)) { *failed = 1; break; }
                mbar_expect_tx(x_full + 8 * stage, N * 128);
                tma_load_2d(smem_u32(base) + stage * STAGE, &tm_x, x_full + 8 * stage, ch * 64, r0);
                if (++stage == STAGES) { stage = 0; parity ^= 1; }
            }
            // (the block does not leave, or use the stages for something else, while a copy is under way)
            for (int i = max(0, asked - STAGES); i < asked; ++i) mbar_wait(x_full + 8 * (i % STAGES), (i / STAGES) & 1);
        }
        __syncwarp();
        __syncthreads();
    } else {
        const bool leader = elect_lane();
        // float accumulate, bf16 x bf16, both K-major, N rows of x, 128 features (tcgen05.cuh: umma_desc)
        const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(N >> 3) << 17) | ((unsigned)(I4T_FEATURES >> 4) << 24);
        const unsigned high = (1024u >> 4) | 1u << 14 | 2u << 29, low = ((smem_u32(base) >> 4) & 0x3FFF) | 1u << 16;
        int stage = 0, parity = 0;
        bool ok = true;
        for (int ch = from; ch < upto; ++ch) {
            if (give_up || !mbar_wait_warp(full + 8 * stage, parity) || !mbar_wait_warp(x_full + 8 * stage, parity)) { ok = false; break; }
            tc5_fence_after();
            const unsigned a = tmem + N + 32 * stage, b = low + stage * (STAGE >> 4);
            if (leader) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    i4t_mma(tmem, a + 8 * k, (unsigned long long)high << 32 | (b + 2 * k), idesc, (ch > from || k > 0) ? 1u : 0u);
                umma_commit(empty + 8 * stage);
            }
            __syncwarp();
            if (++stage == STAGES) { stage = 0; parity ^= 1; }
        }
        // (after giving up too: the block goes on when the products that were issued have ended)
        if (!ok) *failed = 1;
        if (leader && upto > from) umma_commit(done);
        __syncwarp();
        if (!ok) mbar_wait_warp(done, 0);
        __syncthreads();
    }
    tc5_fence_before();
    __syncthreads();
    if (warp == I4T_LOADERS + 1) {
        tc5_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)COLUMNS) : "memory");
    }
    if (splits > 1) cluster_sync();                // every block's sums are in place
    pdl_wait();                                    // (what is written may still be read)
    {
        constexpr int OUT = GLU ? I4T_FEATURES / 2 : I4T_FEATURES, QUADS = OUT / 4;
        const float* d = reinterpret_cast<const float*>(base);
        const int wide = GLU ? p.n / 2 : p.n, rows_here = min(N, p.rows - r0), items = rows_here * QUADS, mine = (items + splits - 1) / splits;
        // IN pieces of four features at a time, whose sums are asked for together; joined in the order of the blocks
        constexpr int IN = 4;
        const int last = min(items, (rank + 1) * mine);
        for (int i0 = rank * mine + threadIdx.x; i0 < last; i0 += IN * I4T_THREADS) {
            float4 s[IN], u[GLU ? IN : 1];
            auto sums = [&](float4 (&to)[IN], int offset) {
#pragma unroll
                for (int x = 0; x < IN; ++x) {
                    const int i = min(i0 + x * I4T_THREADS, last - 1);
                    const float* at = d + i / QUADS * I4T_FEATURES + i % QUADS * 4 + offset;
                    if (splits == 1) {
                        to[x] = *reinterpret_cast<const float4*>(at);
                    } else {
                        to[x] = cluster_f32x4(cluster_peer(at, 0u));
                    }
                }
                for (int j = 1; j < splits; ++j) {
                    float4 v[IN];
#pragma unroll
                    for (int x = 0; x < IN; ++x) {
                        const int i = min(i0 + x * I4T_THREADS, last - 1);
                        v[x] = cluster_f32x4(cluster_peer(d + i / QUADS * I4T_FEATURES + i % QUADS * 4 + offset, (unsigned)j));
                    }
#pragma unroll
                    for (int x = 0; x < IN; ++x) { to[x].x += v[x].x; to[x].y += v[x].y; to[x].z += v[x].z; to[x].w += v[x].w; }
                }
            };
            sums(s, 0);
            if constexpr (GLU) sums(u, OUT);
#pragma unroll
            for (int x = 0; x < IN; ++x) {
                const int i = i0 + x * I4T_THREADS, row = i / QUADS, feature = block * OUT + i % QUADS * 4;
                if (i >= last || feature >= wide) continue;
                float v[4] = {s[x].x, s[x].y, s[x].z, s[x].w};
                if constexpr (GLU) {
                    v[0] = glu_gate_16(v[0], p.act) * u[x].x; v[1] = glu_gate_16(v[1], p.act) * u[x].y;
                    v[2] = glu_gate_16(v[2], p.act) * u[x].z; v[3] = glu_gate_16(v[3], p.act) * u[x].w;
                }
                const size_t to = (size_t)(r0 + row) * wide + feature;
                if (!GLU && p.bias) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += feature + e < wide ? p.bias[feature + e] : 0.f;
                }
                if ((wide & 3) == 0) {             // (a whole piece, and aligned)
                    if (!GLU && p.y32) *reinterpret_cast<float4*>(p.y32 + to) = make_float4(v[0], v[1], v[2], v[3]);
                    else *reinterpret_cast<uint2*>(p.y + to) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (feature + e >= wide) break;
                        if (!GLU && p.y32) p.y32[to + e] = v[e];
                        else p.y[to + e] = __float2bfloat16_rn(v[e]);
                    }
                }
            }
        }
    }
    if (splits > 1) cluster_sync();                // nobody reads this block's memory any more
}

template <int N, int GS, bool GLU, bool TRIAL = false>
static int launch_int4_tile(const I4Params& p, cudaStream_t stream) {
    static int ready[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(-101, "int4_linear: cannot tell the current device");
    if (!ready[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(int4_tile_kernel<N, GS, GLU, TRIAL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)I4T_SMEM<N>);
        if (e != cudaSuccess) return fail(-101, "int4_linear: cannot reserve %zu bytes of shared memory: %s", I4T_SMEM<N>, cudaGetErrorString(e));
        ready[dev] = 1;
    }
    const long long blocks = ((p.n + 15) / 16 + 7) / 8;               // (a gated block's eight tile rows are four of each half)
    // Columns shared out while every block has a place at once and at least 8 chunks (12 with 65 to 128 rows); above 128 rows, where what is joined is
    // larger, by 4 at most.  us with 1, 2, 4 and 8 blocks: 2,048 x 2,048, 24 rows 8.5 / 6.6 / 5.5 / 5.4, 64 rows 9.4 / 7.3 / 6.5 / 7.5; 6,144 x 2,048, 64 rows
    // 9.7 / 7.7 / 8.4 / 16.6, 128 rows 11.1 / 8.9 / 12.0 / 23.7; 2,048 x 8,192, 64 rows 32 / 18 / 12 / 11, 256 rows 43 / 26 / 18 / 31; 8,192 x 28,672, 64 rows
    // 141 / 80 / 45.
    const long long all = blocks * ((p.rows + N - 1) / N), held = (long long)sm_count() * I4T_BLOCKS<N>;
    int splits = 1;
    while (splits < (N > 128 ? 4 : 8) && 2 * splits * all <= held && p.chunks / (2 * splits) >= (N == 128 ? 12 : 8)) splits *= 2;
    CUtensorMap tm;
    const int rc = kmajor_map(&tm, "int4_linear", p.x, p.rows, p.k, N, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, false);
    if (rc != 0) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks * splits), (unsigned)((p.rows + N - 1) / N));
    cfg.blockDim = dim3(I4T_THREADS);
    cfg.dynamicSmemBytes = I4T_SMEM<N>;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return check_launch("int4_linear (tcgen05)", cudaLaunchKernelEx(&cfg, int4_tile_kernel<N, GS, GLU, TRIAL>, tm, p, splits));
}

template <int GS>
static int int4_tile(const I4Params& p, bool glu, cudaStream_t stream) {
    if (p.rows <= 32) return glu ? launch_int4_tile<32, GS, true>(p, stream) : launch_int4_tile<32, GS, false>(p, stream);
    if constexpr (GS == 4)                         // (one form of the kernel has the trial)
        if (p.trial >= 0 && p.rows <= 64) return glu ? launch_int4_tile<64, GS, true, true>(p, stream) : launch_int4_tile<64, GS, false, true>(p, stream);
    if (p.rows <= 64) return glu ? launch_int4_tile<64, GS, true>(p, stream) : launch_int4_tile<64, GS, false>(p, stream);
    if (p.rows <= 128) return glu ? launch_int4_tile<128, GS, true>(p, stream) : launch_int4_tile<128, GS, false>(p, stream);
    return glu ? launch_int4_tile<256, GS, true>(p, stream) : launch_int4_tile<256, GS, false>(p, stream);
}

}  // namespace vapi
