// Attention of prompt portions over an 8-bit cache on the fifth-generation tensor cores (tcgen05): bfloat16 queries, head size 64
// or 128, sequences that bring at least `min_q` tokens to the step (shorter ones are decode8_kernel's).
//
// A block owns twice 128 rows (query token, q head of the group) of one (sequence, kv head) and walks the key tiles, 64 keys each, that
// any of them can see; where those blocks would leave multiprocessors without one, up to 8 of a cluster walk a part of the tiles each and
// join what they have (its log-sum form, always in the same order) through one another's shared memory.
//
// What bounds it: the softmax.  256 rows of 64 keys are 16,384 exponentials, 1,024 cycles of a multiprocessor's, and the tile takes 1,950: the
// two softmax warps of a scheduler are mostly in the same phase, and loads of scores, the maximum and the barriers are not hidden behind the other's
// exponentials.  The products take 960 cycles.  2,048 tokens behind 5,952, 32 / 8 heads of 64: 238 us, 492 TFLOP/s (the 16-bit kernel 243);
// head size 128 426.
//
//   warp 12            issues S = Q K^T of either half into one of its two tensor-memory buffers and O += P V into a third; owns the
//                      allocation;
//   warps 0..3         bring the codes of a tile into registers while the tile before is worked on, and write it to a ring of
//                      shared-memory stages as 16-bit numbers, once for both halves (with 128 rows a block, and two blocks a
//                      multiprocessor, this was a third of all instructions), a warp on each of the four schedulers, which have two
//                      of the softmax warps each: with three, those beside them were what the others waited for;
//   warps 4..7, 8..11  softmax of a half, one row a thread, as the 16-bit kernel does it (attention_tc.cuh), but that the running
//                      maximum only moves when a tile exceeds it by more than 2^24: P is bfloat16, whose rounding is the same at
//                      any magnitude, and float sums hold 2^24 times as much.  A rescaling of O waits for P V and costs 1,500
//                      cycles of a tile's 2,000; at 2^8 one tile in seven had one.
//
//   K: a code is an f16 number; Q's rows are f16 too, each scaled by a power of two so that its largest element is near 2^14 (as in
//      cache8_decode.cuh).  The scale of a block of 16 keys multiplies 16 columns of S, where a score is multiplied by something
//      anyway: it costs nothing.
//   V: O is one sum over all tiles, so V must be on one scale; code * 2^e is a bfloat16 number exactly, and P is bfloat16 as in
//      the 16-bit kernel.
//
// Keys that a row does not see are masked by selection, and the values of those that no row of the block sees are written as zeros.  (A NaN among the
// values that some of the block's rows see and others do not can reach the others through 0 * NaN; the step that wrote it was lost.)  Every wait is bounded; a role that
// gives up records status 16 and the block drains (tensor memory is released on every path).
#pragma once
#include "cache8.cuh"
#include "attention_tc.cuh"        // ft_tile
#include "cluster.cuh"
#include <type_traits>

namespace vapi {

constexpr int P8_HALF = 128, P8_HALVES = 2, P8_ROWS = P8_HALF * P8_HALVES, P8_KEYS = 64, P8_LOADERS = 128, P8_THREADS = P8_LOADERS + P8_ROWS + 32;
constexpr int P8_MIN_Q = 32;                       // in a step of several sequences, those with fewer tokens go to decode8_kernel
template <int HD> constexpr int P8_STAGES = HD == 64 ? 4 : 3;                                // (S two tiles ahead of P V: three at least)
template <int HD> constexpr int P8_TILE = P8_KEYS * HD * 2;                                  // bytes of K (or V) of a tile
template <int HD> constexpr size_t P8_SMEM = 1024 + P8_ROWS * HD * 2 + 2 * P8_ROWS * P8_KEYS * 2 + (size_t)P8_STAGES<HD> * 2 * P8_TILE<HD> + 512;
constexpr float P8_RAISE = 24.f;                   // log2 units by which a tile must exceed the running maximum to raise it
constexpr int P8_TMEM_COLS = 512;                  // a half's S0 | S1, the other's, then O of either, HD columns

// 16 codes as 16 halves
__device__ __forceinline__ void p8_halves(const uint4& c, uint4& lo, uint4& hi) {
    const unsigned w[4] = {c.x, c.y, c.z, c.w};
    unsigned h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) c8_halves4(w[i], h[2 * i], h[2 * i + 1]);
    lo = make_uint4(h[0], h[1], h[2], h[3]);
    hi = make_uint4(h[4], h[5], h[6], h[7]);
}
// 16 codes times f as 16 bfloat16
__device__ __forceinline__ void p8_numbers(const uint4& c, float f, uint4& lo, uint4& hi) {
    const unsigned w[4] = {c.x, c.y, c.z, c.w};
    unsigned h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned a, b;
        c8_halves4(w[i], a, b);
        const float2 x = __fmul2_rn(c8_pair(a), make_float2(f, f)), y = __fmul2_rn(c8_pair(b), make_float2(f, f));
        h[2 * i] = pack_bf16(x.x, x.y);
        h[2 * i + 1] = pack_bf16(y.x, y.y);
    }
    lo = make_uint4(h[0], h[1], h[2], h[3]);
    hi = make_uint4(h[4], h[5], h[6], h[7]);
}

// JOIN: whether `splits` blocks of a cluster share a tile's keys.  (A kernel of its own: the registers of the join in the same one cost the
// other 5%.)
template <int HD, bool JOIN>
__global__ void __launch_bounds__(P8_THREADS, 1)
prompt8_kernel(const C8Params p, const __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ out, const int num_seqs, const int min_q,
               const int blocks) {
    constexpr int STAGES = P8_STAGES<HD>, TILE = P8_TILE<HD>, ATOMS = HD / 64, ATOM = P8_KEYS * 128;     // 64 elements of 64 keys
    extern __shared__ unsigned char p8_smem[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(p8_smem) + 1023) & ~(uintptr_t)1023);
    unsigned char* sQ = base;                                   // [half][atom][128 rows][128 B], 128-byte swizzle
    unsigned char* sP = base + P8_ROWS * HD * 2;                // [half][two buffers][128 rows][128 B]
    unsigned char* sKV = sP + 2 * P8_ROWS * P8_KEYS * 2;        // [stage][K | V][atom][64 keys][128 B]
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(sKV + (size_t)STAGES * 2 * TILE);
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + 32);
    int* flags = reinterpret_cast<int*>(tmem_slot + 1);
    float* sE = reinterpret_cast<float*>(tmem_slot + 4);        // [stage][4]: the scales of the tile's blocks of keys
    // for the join of a cluster, where Q, P, K and V were: O [row][piece of 16 bytes], then the rows' maxima and sums
    auto join_at = [&](int r, int piece) { return reinterpret_cast<float*>(base + (size_t)r * HD * 4 + ((piece ^ (r & 7)) << 4)); };
    float* join_m = reinterpret_cast<float*>(base + P8_ROWS * HD * 4);
    float* join_l = join_m + P8_ROWS;
    static_assert(P8_ROWS * HD * 4 + P8_ROWS * 8 <= P8_ROWS * HD * 2 + 2 * P8_ROWS * P8_KEYS * 2 + STAGES * 2 * TILE, "the join fits");

    // (by a shuffle: what depends on the warp alone is then known to be the same for all its lanes)
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int splits = JOIN ? blocks : 1, rank = JOIN ? (int)blockIdx.x % splits : 0, unit = (int)blockIdx.x / splits, g = unit % p.nkv, n_rep = p.nh / p.nkv;
    // index data was copied from the host before the step's first kernel: safe before the wait
    int s = 0, tile = 0;
    if (!ft_tile(p.cu_q, num_seqs, min_q, n_rep, P8_ROWS, unit / p.nkv, s, tile)) {        // (the same for the whole cluster)
        pdl_wait();
        return;
    }
    const int q0 = p.cu_q[s], qlen = p.cu_q[s + 1] - q0, klen = p.seqlens_k[s];
    const int rows_total = qlen * n_rep, tile_start = tile * P8_ROWS;
    const int last_row = min(rows_total, tile_start + P8_ROWS) - 1;
    const int base_pos = klen - qlen;
    const int p_min = base_pos + tile_start / n_rep, p_max = base_pos + last_row / n_rep;
    const int key_lo = p.window > 0 ? max(0, p_min - p.window + 1) : 0;
    const int nt_all = p_max < key_lo ? 0 : p_max / P8_KEYS - key_lo / P8_KEYS + 1;
    const int nt_before = (int)((long long)nt_all * rank / splits), nt = (int)((long long)nt_all * (rank + 1) / splits) - nt_before;
    const int kt_lo = key_lo / P8_KEYS + nt_before;                 // this block's tiles: kt_lo .. kt_lo + nt - 1

    const unsigned kv_full = smem_u32(bars), kv_empty = smem_u32(bars + STAGES);
    // of half h and buffer b: 16 h + 8 b bytes further on
    const unsigned s_full = smem_u32(bars + 2 * STAGES);
    const unsigned p_ready = smem_u32(bars + 2 * STAGES + 4), pv_done = smem_u32(bars + 2 * STAGES + 8);
    const unsigned q_ready = smem_u32(bars + 2 * STAGES + 12);
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(kv_full + 8 * i, P8_LOADERS); mbar_init(kv_empty + 8 * i, 1); }
        for (int i = 0; i < 2 * P8_HALVES; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_ready + 8 * i, P8_HALF);
            mbar_init(pv_done + 8 * i, 1);
        }
        mbar_init(q_ready, P8_ROWS);
        flags[0] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == P8_THREADS / 32 - 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((unsigned)P8_TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    pdl_trigger();                                  // (not before the allocation: a block of the next kernel that came between would be waited for, and wait)
    const unsigned tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);          // half h: S at 128 h (and 64 further on), O at 256 + HD h

    if (warp == P8_THREADS / 32 - 1) {
        {
            // (the whole warp goes through the loop and waits; one lane issues)
            const bool leader = elect_lane();
            // instruction descriptors: float accumulate, N = 64, M = 128; f16 x f16, both K-major, and bf16 x bf16 with V's
            // contiguous dimension N
            const unsigned shape = (1u << 4) | ((unsigned)(P8_KEYS >> 3) << 17) | ((unsigned)(P8_HALF >> 4) << 24);
            const unsigned idesc_s = shape, idesc_o = shape | (1u << 7) | (1u << 10) | (1u << 16);
            bool ok = true;
            // Descriptors are made once (tcgen05.cuh: umma_desc, umma_desc_mn), and a step's is a sum, of numbers that are the same for the
            // whole warp: a product's operands are in uniform registers.  (With one lane alone in the loop each of them was moved there
            // for every product: four products and a commit took 310 cycles to issue and 192 to run, and the waits between them were not
            // hidden: what bounded the kernel.)
            const unsigned high = (1024u >> 4) | 1u << 14 | 2u << 29;
            const unsigned q_low = ((smem_u32(sQ) >> 4) & 0x3FFF) | 1u << 16, p_low = ((smem_u32(sP) >> 4) & 0x3FFF) | 1u << 16;
            const unsigned k_low = ((smem_u32(sKV) >> 4) & 0x3FFF) | 1u << 16, v_low = (((smem_u32(sKV) + TILE) >> 4) & 0x3FFF) | (1024u >> 4) << 16;
            auto desc = [&](unsigned low) { return (unsigned long long)high << 32 | low; };
            auto score = [&](int h, int i, unsigned kb) {        // S(i) of half h
                if (leader) {
#pragma unroll
                    for (int a = 0; a < ATOMS; ++a)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f16(tmem_base + h * 128 + (i & 1) * 64, desc(q_low + (h * P8_HALF * HD * 2 + a * P8_HALF * 128 + k * 32 >> 4)),
                                     desc(kb + (a * ATOM + k * 32 >> 4)), idesc_s, (a > 0 || k > 0) ? 1u : 0u);
                    umma_commit(s_full + 16 * h + 8 * (i & 1));
                }
                __syncwarp();
            };
            // S runs two tiles ahead of P V, so that a half's softmax finds its next scores there: when P(i) of a half is ready, its
            // S(i) has been read too, and O += P(i) V and S(i + 2) follow one another without another wait.
            int ahead = 0, parity = 0;                           // the stage of the next S
            auto next_tile = [&](unsigned& kb) {
                if (!mbar_wait_warp(kv_full + 8 * ahead, parity)) return false;
                tc5_fence_after();
                kb = k_low + ahead * (2 * TILE >> 4);
                if (++ahead == STAGES) { ahead = 0; parity ^= 1; }
                return true;
            };
            unsigned kb = 0;
            if (nt > 0 && !mbar_wait_warp(q_ready, 0)) ok = false;
            for (int i = 0; i < min(nt, 2) && ok; ++i) {
                if (!next_tile(kb)) { ok = false; break; }
                score(0, i, kb);
                score(1, i, kb);
            }
            int stage = 0;
            for (int i = 0; i < nt && ok; ++i) {
                const unsigned vb = v_low + stage * (2 * TILE >> 4);
#pragma unroll
                for (int h = 0; h < P8_HALVES; ++h) {
                    if (!ok || !mbar_wait_warp(p_ready + 16 * h + 8 * (i & 1), (i >> 1) & 1)) { ok = false; break; }
                    tc5_fence_after();
                    const unsigned pa = p_low + (2 * h + (i & 1)) * (P8_HALF * P8_KEYS * 2 >> 4), tO = tmem_base + 256 + h * HD;
                    if (leader) {
#pragma unroll
                        for (int a = 0; a < ATOMS; ++a)
#pragma unroll
                            for (int k = 0; k < P8_KEYS / 16; ++k)
                                umma_f16(tO + a * 64, desc(pa + k * (32 >> 4)), desc(vb + (a * ATOM + k * 16 * 128 >> 4)), idesc_o, (i > 0 || k > 0) ? 1u : 0u);
                        umma_commit(pv_done + 16 * h + 8 * (i & 1));
                    }
                    __syncwarp();
                    if (i + 2 < nt) {
                        if (h == 0 && !next_tile(kb)) { ok = false; break; }
                        score(h, i + 2, kb);
                    }
                }
                if (ok && leader) umma_commit(kv_empty + 8 * stage);
                if (++stage == STAGES) stage = 0;
            }
            if (!ok) flags[0] = 1;
        }
    } else if (warp < 4) {
        // ---- codes to numbers ----
        const int t = threadIdx.x;
        constexpr int PER = 2 * P8_KEYS * HD / 16, EACH = (PER + P8_LOADERS - 1) / P8_LOADERS;       // 16-byte pieces of a tile, a thread
        const int* bt = p.block_table + (size_t)s * p.table_stride;
        const int per_head = p.page_size / C8_BLOCK;
        const int fresh = !p.settled || base_pos < 0 ? 0 : base_pos / C8_BLOCK * C8_BLOCK;      // from here on a kernel not yet waited for may have written
        bool waited = false;
        // Where the 32 blocks of eight tiles lie, one a lane, and their scales.  Looked up in two steps, both well before they are
        // wanted: a tile's codes are asked for two tiles ahead, and waiting for the table first would double the way.
        // Blocks before the window of the block's first row are not looked up either: their pages may have been given back.
        const int first = key_lo / C8_BLOCK * C8_BLOCK;
        auto key_of = [&](int from) { return (kt_lo + from) * P8_KEYS + lane * C8_BLOCK; };
        auto pages = [&](int from) {                             // of tiles from .. from + 7
            const int key = key_of(from);
            return from + (lane >> 2) < nt && key >= first && key <= p_max ? bt[key / p.page_size] : -1;
        };
        auto places = [&](int from, int page) {
            const int key = key_of(from);
            if (!(from + (lane >> 2) < nt && key >= first && key <= p_max)) return 0;             // (no row sees it: any block, and masked)
            if (page < 0 || page >= p.num_pages) {
                if (p.status) atomicExch(p.status, 4);
                page = 0;
            }
            return (page * 2 * p.nkv + g) * per_head + key % p.page_size / C8_BLOCK;
        };
        auto scales_of = [&](int from, int where) {
            if (!waited && (kt_lo + from + 8) * P8_KEYS > fresh) { pdl_wait(); waited = true; }
            return c8_scales(p, where, per_head);
        };
        const size_t to_values = (size_t)p.nkv * per_head * C8_BLOCK * HD;
        int where = 0, scales = 0, next_page = -1, next_where = 0, next_scales = 0;
        struct Tile { uint4 codes[EACH]; int scales; } even, odd;
        auto load = [&](int i, Tile& to) {                       // tile i (one after the other)
            const int at = i & 7;
            if (i > 0 && at == 0) { where = next_where; scales = next_scales; }
            if (at == 3) next_page = pages(i + 5);
            if (at == 5) {
                next_where = places(i + 3, next_page);
                next_scales = scales_of(i + 3, next_where);
            }
            to.scales = __shfl_sync(0xffffffffu, scales, at * 4 + (lane & 3));
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                const int piece = t + j * P8_LOADERS;
                const int kind = piece / (PER / 2), r = piece % (PER / 2) / (HD / 16), c = piece % (HD / 16);
                const int block = __shfl_sync(0xffffffffu, where, at * 4 + (r / C8_BLOCK & 3));
                if (piece < PER)
                    to.codes[j] = __ldcg(reinterpret_cast<const uint4*>(p.codes + (size_t)block * (C8_BLOCK * HD) + (kind ? to_values : 0) + (r & (C8_BLOCK - 1)) * HD) + c);
            }
        };
        auto write = [&](int i, const Tile& from) {
            const int stage = i % STAGES, k0 = (kt_lo + i) * P8_KEYS;
            if (!__all_sync(0xffffffffu, i < STAGES || mbar_wait(kv_empty + 8 * stage, ((i / STAGES) - 1) & 1))) { flags[0] = 1; return false; }
            unsigned char* dst = sKV + (size_t)stage * 2 * TILE;
            if (t < 4) sE[stage * 4 + t] = c8_power((int)(signed char)(from.scales & 0xff));
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                const int piece = t + j * P8_LOADERS;
                const int kind = piece / (PER / 2), r = piece % (PER / 2) / (HD / 16), c = piece % (HD / 16);
                const int e = (int)(signed char)(__shfl_sync(0xffffffffu, from.scales, r / C8_BLOCK & 3) >> 8 & 0xff);
                if (piece >= PER) continue;
                uint4 lo, hi;
                if (kind == 0) {
                    p8_halves(from.codes[j], lo, hi);
                } else if (k0 + r >= key_lo && k0 + r <= p_max) {       // (what no row sees may be anything)
                    p8_numbers(from.codes[j], c8_power(e), lo, hi);
                } else {
                    lo = hi = make_uint4(0u, 0u, 0u, 0u);
                }
                unsigned char* row = dst + kind * TILE + (c >> 2) * ATOM + r * 128;
                const int ch = 2 * (c & 3);
                *reinterpret_cast<uint4*>(row + ((ch ^ (r & 7)) << 4)) = lo;
                *reinterpret_cast<uint4*>(row + (((ch + 1) ^ (r & 7)) << 4)) = hi;
            }
            fence_proxy_async();
            mbar_arrive(kv_full + 8 * stage);
            return true;
        };
        if (nt > 0) {
            where = places(0, pages(0));
            scales = scales_of(0, where);
            load(0, even);
        }
        if (nt > 1) load(1, odd);
        for (int i = 0; i < nt; i += 2) {
            if (!write(i, even)) break;
            if (i + 2 < nt) load(i + 2, even);
            if (i + 1 >= nt || !write(i + 1, odd)) break;
            if (i + 3 < nt) load(i + 3, odd);
        }
        if (!waited) pdl_wait();
    } else {
        // ---- softmax and epilogue: one row per thread ----
        const int half = (warp - 4) >> 2, quarter = warp & 3;       // (a quarter: the tensor-memory lanes this warp may touch)
        const int row = quarter * 32 + lane;
        const unsigned lane_addr = (unsigned)(quarter * 32) << 16;
        const unsigned tS0 = tmem_base + half * 128, tO = tmem_base + 256 + half * HD;
        const unsigned my_full = s_full + 16 * half, my_ready = p_ready + 16 * half, my_done = pv_done + 16 * half;
        unsigned char* const myP = sP + half * 2 * P8_HALF * P8_KEYS * 2;
        const int start = tile_start + half * P8_HALF;
        const int rr = start + row;
        // the least and the largest position of the half's rows (a half without rows: nothing is stored of it)
        const int my_min = base_pos + start / n_rep, my_max = base_pos + min(last_row, start + P8_HALF - 1) / n_rep;
        const bool row_ok = rr < rows_total;
        const int tok = row_ok ? rr / n_rep : 0;
        const int head = g * n_rep + (row_ok ? rr - tok * n_rep : 0);
        const int pos = row_ok ? base_pos + tok : -1;               // -1: sees nothing
        pdl_wait();                                                 // q comes from the kernel before this one
        float row_f;
        {
            const uint4* src = reinterpret_cast<const uint4*>(q + (size_t)(q0 + tok) * p.q_row_stride + (size_t)head * HD);
            uint4 v[HD / 8];
            float big = 0.f;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) v[c] = row_ok ? src[c] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
                const unsigned w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) big = fmaxf(big, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
            }
            const int x = min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 127);
            const float up = c8_power(14 - x);
            row_f = c8_power(x - 14) * p.scale_log2e;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
                const unsigned w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
                unsigned h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = d8_half2(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up);
                *reinterpret_cast<uint4*>(sQ + half * P8_HALF * HD * 2 + (c >> 3) * P8_HALF * 128 + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            }
            fence_proxy_async();
            mbar_arrive(q_ready);
        }
        float m_run = -INFINITY, l_run = 0.f;
        bool ok = true, s_there = false, kv_there = false;
        for (int i = 0; i < nt && ok; ++i) {
            const int sb = i & 1, stage = i % STAGES;
            const int k0 = (kt_lo + i) * P8_KEYS;
            // (a wait's outcome is made uniform over the warp: the tensor-memory accesses below are warp-wide instructions)
            if (!__all_sync(0xffffffffu, s_there) && !__all_sync(0xffffffffu, mbar_wait(my_full + 8 * sb, (i >> 1) & 1))) { ok = false; break; }
            tc5_fence_after();
            float sv[P8_KEYS];
            float4 ek;
            {
                unsigned raw[P8_KEYS / 16][16];                     // all four loads in flight, one wait
#pragma unroll
                for (int j = 0; j < P8_KEYS / 16; ++j) tmem_ld16_nowait(tS0 + sb * 64 + lane_addr + j * 16, raw[j]);
                // (complete already: makes the scales visible here)
                if (!__all_sync(0xffffffffu, kv_there) && !__all_sync(0xffffffffu, mbar_wait(kv_full + 8 * stage, (i / STAGES) & 1))) {
                    ok = false;
                    tmem_ld_wait();
                    break;
                }
                ek = *reinterpret_cast<const float4*>(sE + stage * 4);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < P8_KEYS / 16; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sv[j * 16 + e] = __uint_as_float(raw[j][e]);
            }
            // (kept above zero: a masked score is -inf before it is multiplied)
            const float f[4] = {fmaxf(ek.x * row_f, 1.2e-38f), fmaxf(ek.y * row_f, 1.2e-38f), fmaxf(ek.z * row_f, 1.2e-38f), fmaxf(ek.w * row_f, 1.2e-38f)};

            const bool need_mask = (k0 + P8_KEYS - 1 > my_min) || (p.window > 0 && k0 <= my_max - p.window);
            if (need_mask) {
#pragma unroll
                for (int e = 0; e < P8_KEYS; ++e) {
                    const int kj = k0 + e;
                    const bool vis = kj <= pos && kj < klen && (p.window <= 0 || kj > pos - p.window);
                    sv[e] = vis ? sv[e] : -INFINITY;
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int b = 0; b < 4; ++b) {                           // (four chains: a single one would leave the warps waiting on latency)
                float m4 = sv[16 * b];
#pragma unroll
                for (int e = 1; e < 16; ++e) m4 = fmaxf(m4, sv[16 * b + e]);
                mx = fmaxf(mx, m4 * f[b]);                          // (the scales are positive)
            }
            const bool grow = mx > m_run + P8_RAISE;                // also the first tile with a visible key
            const float m_new = grow ? mx : m_run;
            const float alpha = grow ? ex2_approx(m_run - m_new) : 1.f;         // m_run = -inf: 0
            if (i >= 1 && __any_sync(0xffffffffu, grow)) {
                // the accumulator must be at rest: P.V of the tile before this one has completed
                if (!__all_sync(0xffffffffu, mbar_wait(my_done + 8 * ((i - 1) & 1), ((i - 1) >> 1) & 1))) { ok = false; break; }
                tc5_fence_after();
#pragma unroll
                for (int j = 0; j < HD / 16; ++j) {
                    float o16[16];
                    tmem_ld16(tO + lane_addr + j * 16, o16);
#pragma unroll
                    for (int e = 0; e < 16; ++e) o16[e] *= alpha;
                    tmem_st16(tO + lane_addr + j * 16, o16);
                }
                tmem_st_wait();
            }
            l_run *= alpha;
            m_run = m_new;
            const float m_use = m_run == -INFINITY ? 0.f : m_run;
            // (this tile's P buffer was last read by P.V of the tile two before, which the half's S of this one was issued behind: it has ended)
            const float2 mu2 = make_float2(-m_use, -m_use);
            // (packed sums, and both barriers of the next tile asked before they are wanted, which keeps their 150 cycles each off a row's chain:
            // 2,048 tokens behind 5,952, 32 / 8 heads of 64, in 241 us, 255 without the two)
            float2 rs2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (c == 5) {                                       // (asked now, wanted when these are written)
                    s_there = mbar_ended(my_full + 8 * (sb ^ 1), ((i + 1) >> 1) & 1);
                    kv_there = mbar_ended(kv_full + 8 * ((i + 1) % STAGES), ((i + 1) / STAGES) & 1);
                }
                unsigned w[4];
                const float2 f2 = make_float2(f[c >> 1], f[c >> 1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float2 x = __ffma2_rn(make_float2(sv[c * 8 + 2 * e], sv[c * 8 + 2 * e + 1]), f2, mu2);
                    x = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                    rs2[e & 1] = __fadd2_rn(rs2[e & 1], x);
                    w[e] = pack_bf16(x.x, x.y);
                }
                *reinterpret_cast<uint4*>(myP + sb * P8_HALF * P8_KEYS * 2 + row * 128 + ((c ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            rs2[0] = __fadd2_rn(rs2[0], rs2[1]);
            l_run += rs2[0].x + rs2[0].y;
            fence_proxy_async();
            tc5_fence_before();
            mbar_arrive(my_ready + 8 * sb);
        }
        if (ok && nt > 0 && !__all_sync(0xffffffffu, mbar_wait(my_done + 8 * ((nt - 1) & 1), ((nt - 1) >> 1) & 1))) ok = false;
        tc5_fence_after();
        if constexpr (JOIN) {
            // Every product of the block is awaited by its half, so with both halves here nothing reads Q, P, K or V any more: O goes there,
            // as floats, a row's pieces of 16 bytes turned by the row so that eight rows' stores meet in no bank.
            __syncthreads();
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {
                float o16[16];
                if (nt > 0 && ok) {
                    tmem_ld16(tO + lane_addr + j * 16, o16);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o16[e] = 0.f;
                }
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<float4*>(join_at(half * P8_HALF + row, j * 4 + c)) = make_float4(o16[4 * c], o16[4 * c + 1], o16[4 * c + 2], o16[4 * c + 3]);
            }
            join_m[half * P8_HALF + row] = m_run;
            join_l[half * P8_HALF + row] = l_run;
        } else if (ok) {                                            // (uniform over the warp)
            const float inv = l_run == 0.f ? 0.f : 1.f / l_run;     // a row that sees nothing: zeros
            __nv_bfloat16* o = out + ((size_t)(q0 + tok) * p.nh + head) * HD;
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {
                float o16[16];
                if (nt > 0) {
                    tmem_ld16(tO + lane_addr + j * 16, o16);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o16[e] = 0.f;
                }
                unsigned w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = inv == 0.f ? 0u : pack_bf16(o16[2 * e] * inv, o16[2 * e + 1] * inv);
                if (row_ok) {
                    *reinterpret_cast<uint4*>(o + j * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                    *reinterpret_cast<uint4*>(o + j * 16 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                }
            }
        }
        if (!ok) flags[0] = 1;
    }
    if constexpr (JOIN) {
        if (warp < 4 || warp == P8_THREADS / 32 - 1) __syncthreads();       // (with the softmax warps')
    }
    // (before the cluster's blocks wait for one another: what they hold meanwhile, another kernel's blocks may be waiting for)
    tc5_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && flags[0] && p.status) atomicExch(p.status, 16);
    if (warp == P8_THREADS / 32 - 1) {
        tc5_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((unsigned)P8_TMEM_COLS) : "memory");
    }
    if constexpr (JOIN) {
        cluster_sync();                                             // every block's result is in place
        const auto join = [&](auto blocks) {
            constexpr int C = decltype(blocks)::value;
            // (a block joins rows that follow one another: neighbours' reads of another block's memory are then one; with every C-th piece
            // a block, 64 KB took 6 us)
            constexpr int MINE = P8_ROWS / C * (HD / 8);
            for (int i = rank * MINE + threadIdx.x; i < (rank + 1) * MINE; i += P8_THREADS) {
                const int r = i / (HD / 8), c = i % (HD / 8), at = tile_start + r;
                if (at >= rows_total) break;
                // (everything is asked for before any of it is used: one after the other, 8 blocks' took 10 us)
                float m[C], l[C], big = -INFINITY, sum = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                float4 o[C][2];
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    m[j] = cluster_f32(cluster_peer(join_m + r, (unsigned)j));
                    l[j] = cluster_f32(cluster_peer(join_l + r, (unsigned)j));
                    o[j][0] = cluster_f32x4(cluster_peer(join_at(r, 2 * c), (unsigned)j));
                    o[j][1] = cluster_f32x4(cluster_peer(join_at(r, 2 * c + 1), (unsigned)j));
                }
#pragma unroll
                for (int j = 0; j < C; ++j) big = fmaxf(big, m[j]);
                const float used = big == -INFINITY ? 0.f : big;
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    const float f = ex2_approx(m[j] - used);
                    const float4 a = o[j][0], b = o[j][1];
                    sum = fmaf(l[j], f, sum);
                    x[0] = fmaf(a.x, f, x[0]); x[1] = fmaf(a.y, f, x[1]); x[2] = fmaf(a.z, f, x[2]); x[3] = fmaf(a.w, f, x[3]);
                    x[4] = fmaf(b.x, f, x[4]); x[5] = fmaf(b.y, f, x[5]); x[6] = fmaf(b.z, f, x[6]); x[7] = fmaf(b.w, f, x[7]);
                }
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                unsigned w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = inv == 0.f ? 0u : pack_bf16(x[2 * e] * inv, x[2 * e + 1] * inv);
                const int token = at / n_rep;
                *reinterpret_cast<uint4*>(out + ((size_t)(q0 + token) * p.nh + g * n_rep + (at - token * n_rep)) * HD + c * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        };
        if (splits == 2) join(std::integral_constant<int, 2>());
        else if (splits == 4) join(std::integral_constant<int, 4>());
        else join(std::integral_constant<int, 8>());
        cluster_sync();                                             // nobody reads this block's memory any more
    }
}

// The limits that a device has to allow, asked once per device, and how many blocks of clusters of 1, 2, 4 and 8 it holds at a time.
template <int HD>
static int prompt8_ready(const int** slots) {
    static int held[64][4];
    static bool ready[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(-101, "paged_attention8: cannot tell the current device");
    if (!ready[dev]) {
        cudaError_t e = cudaFuncSetAttribute(prompt8_kernel<HD, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P8_SMEM<HD>);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(prompt8_kernel<HD, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P8_SMEM<HD>);
        if (e != cudaSuccess) return fail(-101, "paged_attention8: cannot reserve %zu bytes of shared memory: %s", P8_SMEM<HD>, cudaGetErrorString(e));
        for (int i = 0; i < 4; ++i) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(8u << i);
            cfg.blockDim = dim3(P8_THREADS);
            cfg.dynamicSmemBytes = P8_SMEM<HD>;
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 1u << i;
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            int clusters = 0;
            if (cudaOccupancyMaxActiveClusters(&clusters, prompt8_kernel<HD, true>, &cfg) != cudaSuccess) {
                cudaGetLastError();
                clusters = 0;
            }
            held[dev][i] = clusters << i;
        }
        ready[dev] = true;
    }
    *slots = held[dev];
    return 0;
}

// How many blocks share the keys of a tile of rows, and how long the step then takes, in microseconds: rounds of blocks, each of a time a key
// tile and one beside (start, Q, the last stores; in a cluster its blocks' wait for one another and the join).  32 / 8 heads of 64, us with 1, 2, 4
// and 8 blocks: 64 tokens behind 3,936 75 / 44 / 28 / 22; 256 behind 3,744 76 / 44 / 30 / 67; 512 behind 3,488 76 / 44 / 59 / 113; 2,048 behind
// 5,952 238 / 279 / 341 / 520.  Head size 128: 128 behind 3,872 124 / 71 / 44 / 69; 1,024 behind 2,976 125 / 130 / 176 / 314.
template <int HD>
static int p8_splits(long long units, int tiles, const int* slots, float& least) {
    const float tile = HD == 64 ? 1.05f : 1.85f, size = HD == 64 ? 1.f : 1.5f;
    int best = 1;
    for (int i = 0; i < 4; ++i) {
        const int c = 1 << i, held = slots[i] > 0 ? slots[i] : 1;
        if (i > 0 && (slots[i] < c || tiles < 2 * c)) break;
        const float time = (float)((units * c + held - 1) / held) * ((float)((tiles + c - 1) / c) * tile + (i == 0 ? 7.f : (8.f + c / 2) * size));
        if (i == 0 || time < least) { best = c; least = time; }
    }
    return best;
}
// the same of a step: n tokens of sequences with at most max_k keys
template <int HD>
static int p8_step(const C8Params& p, int n, int max_k, float& time) {
    time = INFINITY;
    const int* slots = nullptr;
    if (prompt8_ready<HD>(&slots) != 0) return 1;
    const int n_rep = p.nh / p.nkv;
    const long long units = ((long long)n * n_rep + P8_ROWS - 1) / P8_ROWS * p.nkv;
    const long long seen = (long long)p.window + P8_ROWS / n_rep, keys = p.window > 0 && seen < max_k ? seen : max_k;
    return p8_splits<HD>(units, (int)((keys + P8_KEYS - 1) / P8_KEYS), slots, time);
}

template <int HD>
static int launch_prompt8(const C8Params& p, const void* q, void* out, int n, int num_seqs, int max_q, int max_k, int min_q, int splits, cudaStream_t stream) {
    const int* slots = nullptr;
    const int rc = prompt8_ready<HD>(&slots);
    if (rc != 0) return rc;
    // tiles of all sequences together: at most those of n tokens in one piece and a ragged one a sequence of at least min_q tokens
    const int n_rep = p.nh / p.nkv;
    const long long longest = ((long long)max_q * n_rep + P8_ROWS - 1) / P8_ROWS, most = n / min_q < num_seqs ? n / min_q : num_seqs;
    const long long whole = (long long)n * n_rep / P8_ROWS + most, tiles = longest * most < whole ? longest * most : whole;
    if (tiles == 0) return 0;
    float time;
    if (splits <= 0) splits = p8_step<HD>(p, n, max_k, time);
    splits = splits >= 8 ? 8 : splits >= 4 ? 4 : splits >= 2 ? 2 : 1;      // (what the kernel joins)
    if (tiles * p.nkv * splits > 0x7fffffffLL) return fail(-1, "paged_attention8: the step exceeds the grid (%lld row tiles, %d kv heads)", tiles, p.nkv);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * p.nkv * splits));
    cfg.blockDim = dim3(P8_THREADS);
    cfg.dynamicSmemBytes = P8_SMEM<HD>;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return check_launch("paged_attention8 (tcgen05)", cudaLaunchKernelEx(&cfg, splits > 1 ? prompt8_kernel<HD, true> : prompt8_kernel<HD, false>, p,
                                                                         (const __nv_bfloat16*)q, (__nv_bfloat16*)out, num_seqs, min_q, splits));
}

}  // namespace vapi
