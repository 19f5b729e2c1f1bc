// Products with 4-bit weights, y = x W^T: W's numbers are (code - zero) * scale, code and zero in 0..15, scale (bfloat16) and zero for
// each group of 32, 64 or 128 columns of a row.
//
// How a weight is laid out (int4_pack in ops/int4.py): tiles of 16 rows x 64 columns, 512 bytes each, a row of tiles in one piece.
// Within a tile lane l of a warp has 16 bytes, a word for each 16 columns: of rows l/4 and l/4 + 8 columns 2 (l & 3), + 1, + 8 and + 9, that is
// the A operands of one mma.sync m16n8k16 (and a store's to tensor memory, int4_tile.cuh).  A pair of codes stands 16 bits apart, so
// that one logical operation makes two bfloat16 of it: 0x4300 | code is 128 + code.  Taking 128 + zero off is exact, and so is the product
// of what is left (-15 .. 15) with a bfloat16; a group's sum is a float and is multiplied by the scale in float.  Nothing is rounded but the
// float sums and the result.
//
// Scales: for each tile row and group (of 32: two for every 64 columns, the last perhaps of nothing) 8 pairs of words, word = scale | (128 + zero) << 16 as two bfloat16, rows l/4 and l/4 + 8.
#include "cluster.cuh"
#include "attention_mma.cuh"       // mma_bf16_16816

using namespace vapi;

constexpr int I4_WARPS = 8;
// Rows of int4_rows_kernel; more go to int4_tile_kernel, which takes the time of 32 for any number up to that.  us of the one and of the other: 2,048 x
// 2,048, 16 rows 3.5 / 5.4, 24 rows 5.3 / 5.5; 6,144 x 2,048 5.3 / 6.5 and 7.5 / 6.8; 16,384 x 2,048 gated 9.0 / 9.8 and 11.8 / 10.0; 2,048 x 8,192 7.5 / 8.4
// and 9.8 / 8.6; 1,536 x 6,912 6.4 / 7.5 and 8.7 / 7.7.
constexpr int I4_MOST_ROWS = 16;
constexpr int I4_TILE_WORDS = 128;                 // 16 x 64 codes

struct I4Params {
    const unsigned* codes; const unsigned* scales;
    int n, k, group;                               // features, columns, columns a scale
    int chunks;                                    // 64 columns each
    const __nv_bfloat16* x; int rows;              // [rows][k]
    const float* bias;
    __nv_bfloat16* y;                              // [rows][n], or [rows][n / 2] for a gated product
    float* y32;                                    // instead of y
    int act;
    int trial;                                     // a rank whose blocks give up at their first wait, or -1
};

// two codes, `shift` and 16 + shift bits up, less their row's zero
__device__ __forceinline__ unsigned i4_pair(unsigned w, int shift, __nv_bfloat162 zero) {
    unsigned u;                                    // (one operation: the two constants in registers)
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(u) : "r"(w >> shift), "r"(0x000f000fu), "r"(0x43004300u));
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), zero);
    return *reinterpret_cast<const unsigned*>(&d);
}
__device__ __forceinline__ __nv_bfloat162 i4_zero(unsigned w) {
    const unsigned u = __byte_perm(w, w, 0x3232);
    return *reinterpret_cast<const __nv_bfloat162*>(&u);
}
__device__ __forceinline__ float i4_scale(unsigned w) { return __uint_as_float(w << 16); }

// four 8 x 8 pieces of 16-bit numbers, a row's address a lane: the B operands of two k-steps
__device__ __forceinline__ uint4 i4_pieces(unsigned addr) {
    uint4 v;
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

#include "int4_tile.cuh"

// ---- few rows -------------------------------------------------------------------------------------
// A block owns WN tile rows (16 features each; for a gated product half of them the gate's and half up's) and 8 NT rows of x; its eight
// warps are WN tile rows x 8 / WN slices of the block's columns, and the blocks of a cluster share out the columns further.
// Weights and scales go from memory to registers, AHEAD tiles of a warp under way; those that it asks for first do not wait for the
// kernel before (weights are nobody's output).  x comes to shared memory once a block, a segment of columns at a time, for all its
// warps: with 8 NT rows, x is NT / 4 times as many bytes a column as a tile row's weights, and read for every tile row alone it
// would be most of the traffic.  Partial results are added in the order of slices, then of blocks.
constexpr int I4_PART = 8 * 16;                    // rows of partial results: eight warps x 16 features

constexpr int I4_SEG = 32, I4_AHEAD = 6;           // tiles of columns of x that shared memory holds at most; tiles of weights under way

template <int NT, int GS, bool GLU>                // GS: k-steps of 16 columns a group (2, 4, 8)
__global__ void __launch_bounds__(I4_WARPS * 32, 2)
int4_rows_kernel(const I4Params p, const int splits, const int wn, const int seg) {
    constexpr int AHEAD = I4_AHEAD, CPG = GS > 4 ? GS / 4 : 1, GPC = GS < 4 ? 4 / GS : 1;      // tiles a group; groups a tile
    extern __shared__ __align__(128) unsigned char i4_smem[];
    float (*part)[8 * NT + 1] = reinterpret_cast<float (*)[8 * NT + 1]>(i4_smem);
    __nv_bfloat16* sx = reinterpret_cast<__nv_bfloat16*>(i4_smem + ((I4_PART * (8 * NT + 1) * 4 + 127) & ~127));
    constexpr int PITCH = I4_SEG * 64;         // (a row's pieces of 16 bytes are turned by the row, so that eight rows' are in unlike banks)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int rank = (int)blockIdx.x % splits, block = (int)blockIdx.x / splits, r0 = blockIdx.y * 8 * NT;
    const int tiles = (p.n + 15) / 16, groups = GS < 4 ? p.chunks * GPC : p.k / p.group;
    const int tn = warp % wn, tk = warp / wn, wk = I4_WARPS / wn;
    pdl_trigger();
    // this warp's tile row: a gated block has wn / 2 of the gate and the same of up
    const int half = wn / 2;
    const int mine = GLU ? (tn < half ? block * half + tn : tiles / 2 + block * half + tn - half) : block * wn + tn;
    const bool real = GLU ? block * half + tn % half < tiles / 2 : mine < tiles;
    const int t = real ? mine : 0;
    // (a group's columns stay with one warp)
    const int whole = (p.chunks + CPG - 1) / CPG;
    const int from = (int)((long long)whole * rank / splits) * CPG, upto = min(p.chunks, (int)((long long)whole * (rank + 1) / splits) * CPG);

    float total[NT][4], sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) total[n][i] = sum[n][i] = 0.f;

    const uint4* codes = reinterpret_cast<const uint4*>(p.codes) + (size_t)t * p.chunks * 32 + lane;
    const uint2* scales = reinterpret_cast<const uint2*>(p.scales) + (size_t)t * groups * 8 + g;
    bool waited = false;
    for (int s0 = from; s0 < upto; s0 += seg) {
        const int tiles_here = min(seg, upto - s0), groups_here = (tiles_here + CPG - 1) / CPG;
        const int begin = s0 + groups_here * tk / wk * CPG, end = min(s0 + tiles_here, s0 + groups_here * (tk + 1) / wk * CPG);
        uint4 w[AHEAD];
        uint2 sc[AHEAD][GPC];
        const uint4* wp = codes + (size_t)begin * 32;
        const uint2* sp = scales + (size_t)(GS < 4 ? begin * GPC : begin / CPG) * 8;
        auto bring = [&](int ch, uint4& to, uint2 (&ts)[GPC]) {            // tile after tile; nothing behind the last is used
            if (ch < end) {
                to = __ldg(wp);
#pragma unroll
                for (int i = 0; i < GPC; ++i) ts[i] = __ldg(sp + 8 * i);
            }
            wp += 32;
            if (CPG == 1 || (ch & 1)) sp += 8 * GPC;
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) bring(begin + i, w[i], sc[i]);
        if (!waited) { pdl_wait(); waited = true; }
        else __syncthreads();                      // (the segment before is read)
        {
            // a warp has every eighth row, a lane every 32nd 16 bytes of it
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int row = 8 * n + warp;
                const bool ok = r0 + row < p.rows;
                const __nv_bfloat16* src = p.x + (ok ? (size_t)(r0 + row) * p.k : 0) + s0 * 64;
                for (int i = lane * 8; i < tiles_here * 64; i += 256) {
                    const bool in = ok && s0 * 64 + i < p.k;
                    cp_async_16(sx + row * PITCH + (i ^ (row & 7) << 3), in ? src + i : p.x, in ? 16 : 0);
                }
            }
            cp_async_commit();
            cp_async_wait<0>();
        }
        __syncthreads();
        // a lane's address in four 8 x 8 pieces of x: eight rows, 32 columns
        unsigned xr = (unsigned)__cvta_generic_to_shared(sx + (lane & 7) * PITCH + (begin - s0) * 64) + (((lane >> 3) ^ (lane & 7)) << 4);
        for (int base = begin; base < end; base += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int ch = base + i;
                if (ch >= end) break;
                uint4 xa[NT], xb[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    xa[n] = i4_pieces(xr + n * 8 * PITCH * 2);
                    xb[n] = i4_pieces((xr ^ 64) + n * 8 * PITCH * 2);
                }
                xr += 128;
                const unsigned words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int q = 0; q < GPC; ++q) {
                    const uint2 s = sc[i][q];
                    const __nv_bfloat162 z0 = i4_zero(s.x), z1 = i4_zero(s.y);
#pragma unroll
                    for (int j = q * (GPC == 1 ? 4 : GS); j < (q + 1) * (GPC == 1 ? 4 : GS); ++j) {
                        const unsigned a[4] = {i4_pair(words[j], 0, z0), i4_pair(words[j], 4, z1), i4_pair(words[j], 8, z0), i4_pair(words[j], 12, z1)};
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const unsigned b[8] = {xa[n].x, xa[n].y, xa[n].z, xa[n].w, xb[n].x, xb[n].y, xb[n].z, xb[n].w};
                            mma_bf16_16816(sum[n], a, b[2 * j], b[2 * j + 1]);
                        }
                    }
                    // a group is complete: its sum on its scale
                    if (GS <= 4 || (ch + 1) % CPG == 0 || ch + 1 == end) {
                        const float f0 = i4_scale(s.x), f1 = i4_scale(s.y);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            total[n][0] = fmaf(sum[n][0], f0, total[n][0]);
                            total[n][1] = fmaf(sum[n][1], f0, total[n][1]);
                            total[n][2] = fmaf(sum[n][2], f1, total[n][2]);
                            total[n][3] = fmaf(sum[n][3], f1, total[n][3]);
                            sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
                        }
                    }
                }
                bring(ch + AHEAD, w[i], sc[i]);
            }
        }
    }
    if (!waited) pdl_wait();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float* lo = part[(tk * wn + tn) * 16 + g], *hi = part[(tk * wn + tn) * 16 + g + 8];
        lo[8 * n + 2 * c] = total[n][0];
        lo[8 * n + 2 * c + 1] = total[n][1];
        hi[8 * n + 2 * c] = total[n][2];
        hi[8 * n + 2 * c + 1] = total[n][3];
    }
    __syncthreads();
    const int features = wn * 16;                  // of the block, with up's behind the gate's (a power of two)
    if (splits > 1) {
        // the block's own sum first, then the cluster's
        if (wk > 1) {
            for (int i = threadIdx.x; i < features * 8 * NT; i += I4_WARPS * 32) {
                const int f = i & (features - 1), n = i >> (31 - __clz(features));
                float s = 0.f;
                for (int k = 0; k < wk; ++k) s += part[k * features + f][n];
                part[f][n] = s;
            }
        }
        cluster_sync();
    }
    // one result (a pair for a gated product) a thread, features side by side
    const int wide = GLU ? p.n / 2 : p.n, mine_f = GLU ? features / 2 : features, rows_here = min(8 * NT, p.rows - r0), shift = 31 - __clz(mine_f);
    for (int i = threadIdx.x * splits + rank; i < mine_f * rows_here; i += I4_WARPS * 32 * splits) {
        const int n = i >> shift, f = i & (mine_f - 1), feature = block * mine_f + f;
        float v[GLU ? 2 : 1];
#pragma unroll
        for (int h = 0; h < (GLU ? 2 : 1); ++h) {
            const int at = f + h * mine_f;
            float s = 0.f;
            if (splits > 1) {
                float peer[8];                     // (all under way together)
#pragma unroll
                for (int j = 0; j < 8; ++j) peer[j] = j < splits ? cluster_f32(cluster_peer(&part[at][n], (unsigned)j)) : 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) s += peer[j];
            } else {
                for (int k = 0; k < wk; ++k) s += part[k * features + at][n];
            }
            v[h] = s;
        }
        if (feature >= wide) continue;
        const size_t to = (size_t)(r0 + n) * wide + feature;
        if (GLU) {
            p.y[to] = __float2bfloat16_rn(glu_gate_16(v[0], p.act) * v[GLU ? 1 : 0]);
        } else {
            const float s = v[0] + (p.bias ? p.bias[feature] : 0.f);
            if (p.y32) p.y32[to] = s;
            else p.y[to] = __float2bfloat16_rn(s);
        }
    }
    if (splits > 1) cluster_sync();                // nobody reads this block's memory any more
}

// How the work falls to blocks: as many tile rows a block (1, 2, 4 or 8) as leave about two blocks a multiprocessor, and for more than 8 rows two where
// K is long, so that x is not read more often than the weights (of a short K, blocks are worth more: 16 rows, one tile row a block or two, 2,048 x
// 2,048 3.8 / 4.5 us, 2,048 x 8,192 8.5 / 7.4); then, while there are fewer blocks, a cluster of up to 8 shares the columns as long as each
// warp still has four tiles.
static void int4_shape(int tiles, int chunks, int nt, bool glu, int& wn, int& splits) {
    const int least = nt > 1 && chunks > 48 ? 2 : 1;
    wn = glu ? 2 : 1;
    while (wn < 8 && (wn < least || (tiles + wn - 1) / wn > 2 * sm_count())) wn *= 2;
    const long long blocks = (tiles + wn - 1) / wn;
    splits = 1;
    while (splits < 8 && 2 * splits * blocks <= 2LL * sm_count() && chunks / (2 * splits * (I4_WARPS / wn)) >= 4) splits *= 2;
}

template <int NT, int GS, bool GLU>
static int launch_int4_rows(const I4Params& p, cudaStream_t stream) {
    const int tiles = (p.n + 15) / 16;
    int wn, splits;
    int4_shape(tiles, p.chunks, NT, GLU, wn, splits);
    const int each = (p.chunks + splits - 1) / splits + 1, seg = (each < I4_SEG ? each + (each & 1) : I4_SEG);
    constexpr size_t smem = ((I4_PART * (8 * NT + 1) * 4 + 127) & ~127) + (size_t)8 * NT * I4_SEG * 64 * 2;
    static int ready[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(-101, "int4_linear: cannot tell the current device");
    if (!ready[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(int4_rows_kernel<NT, GS, GLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail(-101, "int4_linear: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
        ready[dev] = 1;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((tiles + wn - 1) / wn * splits), (unsigned)((p.rows + 8 * NT - 1) / (8 * NT)));
    cfg.blockDim = dim3(I4_WARPS * 32);
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
    return check_launch("int4_linear", cudaLaunchKernelEx(&cfg, int4_rows_kernel<NT, GS, GLU>, p, splits, wn, seg));
}

template <int GS>
static int int4_rows(const I4Params& p, bool glu, cudaStream_t stream) {
    if (p.rows <= 8) return glu ? launch_int4_rows<1, GS, true>(p, stream) : launch_int4_rows<1, GS, false>(p, stream);
    return glu ? launch_int4_rows<2, GS, true>(p, stream) : launch_int4_rows<2, GS, false>(p, stream);
}

// x [rows][k] bfloat16 with 16-byte aligned rows.  gated: W is [gate; up], y [rows][n / 2] = act(gate) * up, n / 2 a multiple of 16.
// y32 instead of y for float32 results (not for a gated product).  trial: -1; from 0 on, with 33 to 64 rows and groups of 64, the rank in its cluster of
// blocks that take no wait.
VAPI_EXPORT int vapi_int4_linear(const void* codes, const void* scales, int n, int k, int group, const void* x, int rows, const float* bias,
                                 void* y, float* y32, int gated, int act, int trial, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (n <= 0 || k <= 0) return fail(-1, "int4_linear: a weight of %d x %d", n, k);
    if (group != 32 && group != 64 && group != 128) return fail(-1, "int4_linear: groups of %d columns are not 32, 64 or 128", group);
    if (k % group != 0) return fail(-1, "int4_linear: %d columns are not a multiple of the group's %d", k, group);
    if (gated && (n % 32 != 0 || bias || y32)) return fail(-1, "int4_linear: a gated product needs a multiple of 32 features (got %d), no bias and bfloat16 results", n);
    if ((((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)x) & 15) != 0) return fail(-1, "int4_linear: an operand is not 16-byte aligned");
    if (rows > 65535 * 128) return fail(-1, "int4_linear: %d rows exceed the grid", rows);
    I4Params p;
    p.codes = (const unsigned*)codes; p.scales = (const unsigned*)scales; p.n = n; p.k = k; p.group = group; p.chunks = (k + 63) / 64;
    p.x = (const __nv_bfloat16*)x; p.rows = rows; p.bias = bias; p.y = (__nv_bfloat16*)y; p.y32 = y32; p.act = act; p.trial = trial;
    if (rows > I4_MOST_ROWS) {
        if (group == 32) return int4_tile<2>(p, gated != 0, stream);
        if (group == 64) return int4_tile<4>(p, gated != 0, stream);
        return int4_tile<8>(p, gated != 0, stream);
    }
    if (group == 32) return int4_rows<2>(p, gated != 0, stream);
    if (group == 64) return int4_rows<4>(p, gated != 0, stream);
    return int4_rows<8>(p, gated != 0, stream);
}

// ---- the weight as numbers --------------------------------------------------------------------------
// A thread takes one word of each of four lanes: 16 columns of two rows.
template <typename T>
__global__ void int4_numbers_kernel(const unsigned* __restrict__ codes, const unsigned* __restrict__ scales, int n, int k, int group, int chunks,
                                    T* __restrict__ out, long long pieces) {
    pdl_trigger();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= pieces) {
        pdl_wait();
        return;
    }
    const int lane = (int)(i & 31), g = lane >> 2, j = lane & 3;
    const int tile = (int)(i / 32 / chunks), col = (int)(i / 32 % chunks) * 64 + 16 * j;
    unsigned words[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) words[c] = __ldg(codes + (i - j + c) * 4 + j);
    const int groups = group == 32 ? 2 * chunks : k / group;
    pdl_wait();                                    // (the weight is nobody's output, but `out` may still be read)
    if (col >= k) return;
    const uint2 sc = __ldg(reinterpret_cast<const uint2*>(scales) + ((size_t)tile * groups + col / group) * 8 + g);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = tile * 16 + g + 8 * h;
        if (row >= n) continue;
        const unsigned s = h ? sc.y : sc.x;
        const float f = i4_scale(s), z = __uint_as_float(s & 0xffff0000u) - 128.f;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            T* dst = out + (size_t)row * k + col + 8 * p;
            float v[8];
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) v[2 * c + e] = ((float)(words[c] >> (8 * p + 4 * h + 16 * e) & 15u) - z) * f;
            if (sizeof(T) == 4) {
                reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                reinterpret_cast<uint4*>(dst)[0] = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
            }
        }
    }
}

// The numbers may become a product's weight, and products take a weight to be nobody's output: they read it before they wait for the kernels ahead of
// them.  So a launch without an early start follows the numbers, which begins when they are in memory and lets nothing begin before it has ended; a
// later kernel's own wait would come too late, and so would that of one in between.  (With the product, us with and without: 8 float32 rows of 16,384 x
// 2,048 66.2 / 64.0, 40 of 2,048 x 8,192 76.9 / 76.3; 2,048 bfloat16 rows of 6,144 x 2,048 47.2 / 46.5.)
__global__ void int4_settled_kernel() {}

// out [n][k], 16-byte aligned
VAPI_EXPORT int vapi_int4_numbers(const void* codes, const void* scales, int n, int k, int group, void* out, int dtype, cudaStream_t stream) {
    if (n <= 0 || k <= 0) return fail(-1, "int4_dequantize: a weight of %d x %d", n, k);
    if ((group != 32 && group != 64 && group != 128) || k % group != 0) return fail(-1, "int4_dequantize: groups of %d of %d columns", group, k);
    if ((((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)out) & 15) != 0) return fail(-1, "int4_dequantize: an operand is not 16-byte aligned");
    const int chunks = (k + 63) / 64;
    const long long pieces = (long long)((n + 15) / 16) * chunks * 32, blocks = (pieces + 255) / 256;
    if (blocks > 0x7fffffffLL) return fail(-1, "int4_dequantize: %d x %d exceeds the grid", n, k);
    cudaError_t e;
    if (dtype == VAPI_F32)
        e = launch(int4_numbers_kernel<float>, (unsigned)blocks, 256, 0, stream, (const unsigned*)codes, (const unsigned*)scales, n, k, group, chunks, (float*)out, pieces);
    else if (dtype == VAPI_BF16)
        e = launch(int4_numbers_kernel<__nv_bfloat16>, (unsigned)blocks, 256, 0, stream, (const unsigned*)codes, (const unsigned*)scales, n, k, group, chunks,
                   (__nv_bfloat16*)out, pieces);
    else
        return fail(-2, "int4_dequantize: unsupported dtype %d", dtype);
    const int rc = check_launch("int4_dequantize", e);
    if (rc != 0) return rc;
    return check_launch("int4_dequantize", launch_if(false, int4_settled_kernel, dim3(1), dim3(32), 0, stream));
}

// ---- a weight laid out -----------------------------------------------------------------------------
// What int4_pack makes of row-major codes, scales and zeros (null: 8 everywhere): a lane a tile's 16 bytes, then a thread a word of scales.  A code or a
// zero above 15 is left in `bad`.
__global__ void int4_pack_kernel(const unsigned char* __restrict__ codes, const unsigned short* __restrict__ scales, const unsigned char* __restrict__ zeros,
                                 int n, int k, int group, int chunks, unsigned* __restrict__ words, unsigned* __restrict__ pairs, long long pieces,
                                 long long all, int* __restrict__ bad) {
    pdl_trigger();
    pdl_wait();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= all) return;
    bool over = false;
    if (i < pieces) {
        const int lane = (int)(i & 31), g = lane >> 2, c = lane & 3, tile = (int)(i / 32 / chunks), ch = (int)(i / 32 % chunks);
        unsigned w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int row = tile * 16 + 8 * h + g, col = ch * 64 + 16 * j + 8 * p + 2 * c;
                    if (row >= n || col >= k) continue;
                    const unsigned x = __ldg(reinterpret_cast<const unsigned short*>(codes + (size_t)row * k + col));
                    over |= (x & 0xf0f0u) != 0u;
                    w[j] |= ((x & 15u) | (x >> 8 & 15u) << 16) << (8 * p + 4 * h);
                }
        reinterpret_cast<uint4*>(words)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        const long long j = i - pieces;            // [tile][group][g][h]
        const int groups = k / group, wide = group == 32 ? 2 * chunks : groups;
        const int h = (int)(j & 1), g = (int)(j >> 1 & 7), at = (int)((j >> 4) % wide), tile = (int)((j >> 4) / wide), row = tile * 16 + 8 * h + g;
        unsigned pair = 0u;
        if (row < n && at < groups) {
            const unsigned z = zeros ? zeros[(size_t)row * groups + at] : 8u;
            over = z > 15u;
            pair = scales[(size_t)row * groups + at] | (0x4300u + (z & 15u)) << 16;      // (128 + zero as bfloat16)
        }
        pairs[j] = pair;
    }
    if (over) atomicExch(bad, 1);
}

// words [tiles][chunks][32][4] and pairs [tiles][groups, or 2 chunks of them][8][2] as int4_pack says; bad: set to 1 or left
VAPI_EXPORT int vapi_int4_pack(const void* codes, const void* scales, const void* zeros, int n, int k, int group, void* words, void* pairs, int* bad,
                               cudaStream_t stream) {
    if (n <= 0 || k <= 0) return fail(-1, "int4_pack: a weight of %d x %d", n, k);
    if ((group != 32 && group != 64 && group != 128) || k % group != 0) return fail(-1, "int4_pack: groups of %d of %d columns", group, k);
    if (((uintptr_t)codes & 7) != 0 || ((uintptr_t)words & 15) != 0) return fail(-1, "int4_pack: the codes are not 8-byte aligned, or the words not 16-byte");
    const int chunks = (k + 63) / 64, tiles = (n + 15) / 16;
    const long long pieces = (long long)tiles * chunks * 32, all = pieces + (long long)tiles * (group == 32 ? 2 * chunks : k / group) * 16, blocks = (all + 255) / 256;
    if (blocks > 0x7fffffffLL) return fail(-1, "int4_pack: %d x %d exceeds the grid", n, k);
    return check_launch("int4_pack", launch(int4_pack_kernel, (unsigned)blocks, 256, 0, stream, (const unsigned char*)codes, (const unsigned short*)scales,
                                            (const unsigned char*)zeros, n, k, group, chunks, (unsigned*)words, (unsigned*)pairs, pieces, all, bad));
}

VAPI_EXPORT const char* vapi_last_error() { return error_buffer(); }
