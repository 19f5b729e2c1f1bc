// Products with 4-bit weights, y = x W^T: W's numbers are (code - zero) * scale, code and zero in 0..15, scale (bfloat16) and zero for
// each group of 32, 64 or 128 columns of a row.
//
// How a weight is laid out (int4_pack in ops/int4.py): tiles of 16 rows x 64 columns, 512 bytes each, a row of tiles in one piece.
// Within a tile lane l of a warp has 16 bytes: rows l/4 and l/4 + 8, columns 8 (l & 3) .. + 7 and 32 + 8 (l & 3) .. + 7, a word four of
// those, that is the A operands of one mma.sync m16n8k16.  A pair of codes stands 16 bits apart, so that one logical operation
// makes two bfloat16 of it: 0x4300 | code is 128 + code.  Taking 128 + zero off is exact, and so is the product of what is left
// (-15 .. 15) with a bfloat16; a group's sum is a float and is multiplied by the scale in float.  Nothing is rounded but the
// float sums and the result.  The order of 32 columns (the smallest group) is free as long as x follows it: a lane's 8 columns of
// x are 16 bytes in one piece, its B operands of two k-steps.
//
// Scales: for each tile row and group 8 pairs of words, word = scale | (128 + zero) << 16 as two bfloat16, rows l/4 and l/4 + 8.
#include "cluster.cuh"
#include "attention_mma.cuh"       // mma_bf16_16816

using namespace vapi;

constexpr int I4_WARPS = 8;
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
};

// two codes, `shift` and 16 + shift bits up, less their row's zero
__device__ __forceinline__ unsigned i4_pair(unsigned w, int shift, __nv_bfloat162 zero) {
    const unsigned u = ((w >> shift) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), zero);
    return *reinterpret_cast<const unsigned*>(&d);
}
__device__ __forceinline__ __nv_bfloat162 i4_zero(unsigned w) {
    const unsigned u = __byte_perm(w, w, 0x3232);
    return *reinterpret_cast<const __nv_bfloat162*>(&u);
}
__device__ __forceinline__ float i4_scale(unsigned w) { return __uint_as_float(w << 16); }

// ---- few rows -------------------------------------------------------------------------------------
// A block owns RT tile rows (16 features each; a gated product's are one of the gate and one of up) and 8 NT rows of x; its
// eight warps, and the blocks of a cluster, share out the columns, 64 at a time.  Weights go from memory to registers, AHEAD tiles of
// each tile row under way; those that a warp asks for first do not wait for the kernel before (weights are nobody's output).
// Partial results are added in warp order, then in block order.
constexpr int I4_AHEAD = 4;

template <int NT, int RT, int GS, bool GLU>        // GS: k-steps of 16 columns a group (2, 4, 8)
__global__ void __launch_bounds__(I4_WARPS * 32, NT == 4 ? 1 : 2)
int4_rows_kernel(const I4Params p, const int splits) {
    __shared__ __align__(16) float part[I4_WARPS][RT][16][8 * NT + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int rank = (int)blockIdx.x % splits, tile = (int)blockIdx.x / splits, r0 = blockIdx.y * 8 * NT;
    const int tiles = (p.n + 15) / 16, groups = p.k / p.group;
    pdl_trigger();
    int t[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) t[r] = GLU ? tile + r * (tiles / 2) : min(tile * RT + r, tiles - 1);
    const int units = splits * I4_WARPS, unit = rank * I4_WARPS + warp;
    // (a group's columns stay with one warp: groups of two tiles are handed out whole)
    constexpr int CPG = GS > 4 ? GS / 4 : 1;       // tiles a group
    const int whole = (p.chunks + CPG - 1) / CPG;
    const int begin = (int)((long long)whole * unit / units) * CPG, end = min(p.chunks, (int)((long long)whole * (unit + 1) / units) * CPG);

    uint4 w[I4_AHEAD][RT];
    auto bring = [&](int ch, uint4 (&to)[RT]) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
            to[r] = ch < end ? __ldg(reinterpret_cast<const uint4*>(p.codes) + ((size_t)t[r] * p.chunks + ch) * 32 + lane) : make_uint4(0u, 0u, 0u, 0u);
    };
#pragma unroll
    for (int i = 0; i < I4_AHEAD; ++i) bring(begin + i, w[i]);
    float total[RT][NT][4], sum[RT][NT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) total[r][n][i] = sum[r][n][i] = 0.f;
    pdl_wait();

    for (int base = begin; base < end; base += I4_AHEAD) {
#pragma unroll
        for (int i = 0; i < I4_AHEAD; ++i) {
            const int ch = base + i;
            if (ch >= end) break;
            // x: 8 and 8 columns of rows g, 8 + g ..
            uint4 xa[NT], xb[NT];
            const int col = ch * 64 + c * 8;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int row = r0 + 8 * n + g;
                const uint4* src = reinterpret_cast<const uint4*>(p.x + (size_t)row * p.k + col);
                const bool ok = row < p.rows;
                xa[n] = ok && col < p.k ? src[0] : make_uint4(0u, 0u, 0u, 0u);
                xb[n] = ok && col + 32 < p.k ? src[4] : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const unsigned words[4] = {w[i][r].x, w[i][r].y, w[i][r].z, w[i][r].w};
#pragma unroll
                for (int part_of = 0; part_of < (GS < 4 ? 4 / GS : 1); ++part_of) {
                    const int group = min(GS < 4 ? ch * 2 + part_of : ch / CPG, groups - 1);      // (columns behind the last: x is zero there)
                    const uint2 sc = __ldg(reinterpret_cast<const uint2*>(p.scales) + ((size_t)t[r] * groups + group) * 8 + g);
                    const __nv_bfloat162 z0 = i4_zero(sc.x), z1 = i4_zero(sc.y);
#pragma unroll
                    for (int j = part_of * GS; j < (GS < 4 ? (part_of + 1) * GS : 4); ++j) {
                        const unsigned a[4] = {i4_pair(words[j], 0, z0), i4_pair(words[j], 4, z1), i4_pair(words[j], 8, z0), i4_pair(words[j], 12, z1)};
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const unsigned b[8] = {xa[n].x, xa[n].y, xa[n].z, xa[n].w, xb[n].x, xb[n].y, xb[n].z, xb[n].w};
                            mma_bf16_16816(sum[r][n], a, b[2 * j], b[2 * j + 1]);
                        }
                    }
                    // a group is complete: its sum on its scale
                    if (GS <= 4 || (ch + 1) % CPG == 0 || ch + 1 == end) {
                        const float s0 = i4_scale(sc.x), s1 = i4_scale(sc.y);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            total[r][n][0] = fmaf(sum[r][n][0], s0, total[r][n][0]);
                            total[r][n][1] = fmaf(sum[r][n][1], s0, total[r][n][1]);
                            total[r][n][2] = fmaf(sum[r][n][2], s1, total[r][n][2]);
                            total[r][n][3] = fmaf(sum[r][n][3], s1, total[r][n][3]);
                            sum[r][n][0] = sum[r][n][1] = sum[r][n][2] = sum[r][n][3] = 0.f;
                        }
                    }
                }
            }
            bring(ch + I4_AHEAD, w[i]);
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            part[warp][r][g][8 * n + 2 * c] = total[r][n][0];
            part[warp][r][g][8 * n + 2 * c + 1] = total[r][n][1];
            part[warp][r][g + 8][8 * n + 2 * c] = total[r][n][2];
            part[warp][r][g + 8][8 * n + 2 * c + 1] = total[r][n][3];
        }
    __syncthreads();
    constexpr int ALL = RT * 16 * 8 * NT;
    if (splits > 1) {
        // the block's own sum first, then the cluster's
        for (int i = threadIdx.x; i < ALL; i += I4_WARPS * 32) {
            const int r = i / (16 * 8 * NT), f = i / (8 * NT) % 16, n = i % (8 * NT);
            float s = 0.f;
#pragma unroll
            for (int v = 0; v < I4_WARPS; ++v) s += part[v][r][f][n];
            part[0][r][f][n] = s;
        }
        cluster_sync();
    }
    // one result (a pair for a gated product) a thread, features side by side
    const int wide = GLU ? p.n / 2 : p.n;
    for (int i = threadIdx.x * splits + rank; i < (GLU ? ALL / 2 : ALL); i += I4_WARPS * 32 * splits) {
        const int n = i / ((GLU ? 1 : RT) * 16), f = i % ((GLU ? 1 : RT) * 16), row = r0 + n;
        const int feature = (GLU ? tile : tile * RT) * 16 + f;
        float v[GLU ? 2 : 1];
#pragma unroll
        for (int h = 0; h < (GLU ? 2 : 1); ++h) {
            const int r = GLU ? h : f / 16;
            float s = 0.f;
            if (splits > 1) {
                for (int j = 0; j < splits; ++j) s += cluster_f32(cluster_peer(&part[0][r][f % 16][n], (unsigned)j));
            } else {
#pragma unroll
                for (int q = 0; q < I4_WARPS; ++q) s += part[q][r][f % 16][n];
            }
            v[h] = s;
        }
        if (row >= p.rows || feature >= wide) continue;
        if (GLU) {
            p.y[(size_t)row * wide + feature] = __float2bfloat16_rn(glu_gate_16(v[0], p.act) * v[GLU ? 1 : 0]);
        } else {
            const float s = v[0] + (p.bias ? p.bias[feature] : 0.f);
            if (p.y32) p.y32[(size_t)row * wide + feature] = s;
            else p.y[(size_t)row * wide + feature] = __float2bfloat16_rn(s);
        }
    }
    if (splits > 1) cluster_sync();                // nobody reads this block's memory any more
}

template <int NT, int RT, int GS, bool GLU>
static int launch_int4_rows(const I4Params& p, int splits, cudaStream_t stream) {
    const int tiles = (p.n + 15) / 16, blocks = GLU ? tiles / 2 : (tiles + RT - 1) / RT;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks * splits), (unsigned)((p.rows + 8 * NT - 1) / (8 * NT)));
    cfg.blockDim = dim3(I4_WARPS * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return check_launch("int4_linear", cudaLaunchKernelEx(&cfg, int4_rows_kernel<NT, RT, GS, GLU>, p, splits));
}

// Blocks of a cluster that share the columns: a power of two up to 8, while there are fewer than two blocks a multiprocessor
// and each warp still has four tiles.
static int int4_splits(long long blocks, int chunks) {
    int s = 1;
    while (s < 8 && 2 * s * blocks <= 2LL * sm_count() && chunks / (2 * s * I4_WARPS) >= 4) s *= 2;
    return s;
}

template <int GS>
static int int4_rows(const I4Params& p, bool glu, cudaStream_t stream) {
    const int tiles = (p.n + 15) / 16;
    // one tile row a block while there are few of them, else two, which halves what is read of x
    const bool two = !glu && tiles >= 4 * sm_count();
    const long long blocks = glu || two ? tiles / 2 : tiles;
    const int splits = int4_splits(blocks, p.chunks);
#define VAPI_I4(NT)                                                                       \
    return glu ? launch_int4_rows<NT, 2, GS, true>(p, splits, stream)                     \
               : two ? launch_int4_rows<NT, 2, GS, false>(p, splits, stream) : launch_int4_rows<NT, 1, GS, false>(p, splits, stream)
    if (p.rows <= 8) VAPI_I4(1);
    if (p.rows <= 16) VAPI_I4(2);
    VAPI_I4(4);
#undef VAPI_I4
}

// x [rows][k] bfloat16 with 16-byte aligned rows.  gated: W is [gate; up], y [rows][n / 2] = act(gate) * up, n / 2 a multiple of 16.
// y32 instead of y for float32 results (not for a gated product).
VAPI_EXPORT int vapi_int4_linear(const void* codes, const void* scales, int n, int k, int group, const void* x, int rows, const float* bias,
                                 void* y, float* y32, int gated, int act, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (n <= 0 || k <= 0) return fail(-1, "int4_linear: a weight of %d x %d", n, k);
    if (group != 32 && group != 64 && group != 128) return fail(-1, "int4_linear: groups of %d columns are not 32, 64 or 128", group);
    if (k % group != 0) return fail(-1, "int4_linear: %d columns are not a multiple of the group's %d", k, group);
    if (gated && (n % 32 != 0 || bias || y32)) return fail(-1, "int4_linear: a gated product needs a multiple of 32 features (got %d), no bias and bfloat16 results", n);
    if ((((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)x) & 15) != 0) return fail(-1, "int4_linear: an operand is not 16-byte aligned");
    if (rows > 65535 * 32) return fail(-1, "int4_linear: %d rows exceed the grid", rows);
    I4Params p;
    p.codes = (const unsigned*)codes; p.scales = (const unsigned*)scales; p.n = n; p.k = k; p.group = group; p.chunks = (k + 63) / 64;
    p.x = (const __nv_bfloat16*)x; p.rows = rows; p.bias = bias; p.y = (__nv_bfloat16*)y; p.y32 = y32; p.act = act;
    if (group == 32) return int4_rows<2>(p, gated != 0, stream);
    if (group == 64) return int4_rows<4>(p, gated != 0, stream);
    return int4_rows<8>(p, gated != 0, stream);
}

// ---- the weight as numbers --------------------------------------------------------------------------
// A thread's 16 bytes are twice 8 columns of two rows.
template <typename T>
__global__ void int4_numbers_kernel(const unsigned* __restrict__ codes, const unsigned* __restrict__ scales, int n, int k, int group, int chunks,
                                    T* __restrict__ out, long long pieces) {
    pdl_trigger();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= pieces) {
        pdl_wait();
        return;
    }
    const int lane = (int)(i & 31), g = lane >> 2, c = lane & 3;
    const int tile = (int)(i / 32 / chunks), ch = (int)(i / 32 % chunks);
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(codes) + i);
    const unsigned words[4] = {w.x, w.y, w.z, w.w};
    const int groups = k / group;
    pdl_wait();                                    // (the weight is nobody's output, but `out` may still be read)
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const int col = ch * 64 + 32 * a + 8 * c;
        if (col >= k) break;
        const uint2 sc = __ldg(reinterpret_cast<const uint2*>(scales) + ((size_t)tile * groups + col / group) * 8 + g);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = tile * 16 + g + 8 * h;
            if (row >= n) continue;
            const unsigned s = h ? sc.y : sc.x;
            const float f = i4_scale(s), z = __uint_as_float(s & 0xffff0000u) - 128.f;
            T* dst = out + (size_t)row * k + col;
            float v[8];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)        // columns 4j + 2p + e: bits from 8p + 4h + 16e on of word 2a + j
                    v[4 * j + e] = ((float)(words[2 * a + j] >> (8 * (e >> 1) + 4 * h + 16 * (e & 1)) & 15u) - z) * f;
            if (sizeof(T) == 4) {
                reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                reinterpret_cast<uint4*>(dst)[0] = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
            }
        }
    }
}

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
    return check_launch("int4_dequantize", e);
}

VAPI_EXPORT const char* vapi_last_error() { return error_buffer(); }
