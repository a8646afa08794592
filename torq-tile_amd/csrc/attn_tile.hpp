// Attention of many rows: tiles of 32 rows a wave, 32 NW a workgroup, against 64 keys at a time. A row is a
// (token, query head) pair of one key head, so the heads of a group share the keys that a tile reads.
//
// Bound by the matrix cores and the vector instructions together: 4 d flops per row and key, and an exponential
// with five operations around it. A wave's tile takes about 1000 cycles of vector instructions, and 1024 (d 128)
// or 512 (d 64) of the matrix cores. A wave issues in order, so the exponentials stand between the products with
// the keys, and the next tile's maximum between those with the values. Two waves a SIMD at d 128 overlap
// them to 1860 cycles a tile, at the clock that the power limit leaves (a prompt of 8192, bf16, 32 / 8 heads:
// 559-585 us, 940-980 TFLOP/s, where the library's 8192^3 product has 1155), three at d 64 to 1050.
//
// As in the few-row kernel the first product is S^T = K Q^T, so a lane holds 32 of a tile's 64 scores of one row
// (its neighbour 32 lanes on holds the others), the statistics are one value a lane, and P^T is the second
// operand of O^T = V^T P^T without leaving the registers. K and V go from memory to LDS directly (16 bytes a
// lane, a tile ahead of their use, two stages; K one tile further), keys past the end and pages that are not
// kept from a block of zeros; int8 rows through registers, where they become 16-bit whole numbers. Their decoding and
// scales stand beside the exponentials (prompts of 4096 at d 64 / 128 / 256: 165 / 220 / 514 us, 106 / 168 / 360
// over 16-bit caches).
//
// Trees: tiles over the context see all of it and are as any other; those that the mask reaches read its words, a
// row's 64 bits a tile. 16 trees of 26 to 62 tokens over 4096-16384 keys (int8, 32 / 8 heads of 128; 120 GFLOP) take 295-301
// us, 11 of join among them, in equal spans of each sequence's own (attn_even_parts), 397-416 in spans of one size. A
// workgroup takes 3.3 us for 64 keys with a CU to itself and 3.9 beside another one, and the 2796 rows fill 3712.
//
// LDS layout of a tile: [key / 16][piece / 4][key % 16][4 pieces of 16 bytes], so that each lane of the 1 KB load
// that fills one [16][4] block has the same key in all of its loads, and looks up one page per tile. A key's
// pieces are at piece ^ f(key), f = 2 bit1(key) + bit2(key): the 8 keys that a 16-byte read of K takes at a
// time and the 4 keys x 32 bytes of a column read of V each cover all 32 banks once.
#pragma once

#include "attn_common.hpp"

namespace tqt {
namespace {

__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The workgroup's sequence and tile among all of the batch's: tiles of a sequence are taken from its last
// rows on, which see the most keys.
__device__ __forceinline__ bool attn_find_tile(const AttnArgs &a, int index, int m, int &b, int &tile, AttnSeq &s)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const bool in = b0 + lane < a.batch;
        const AttnSeq mine = attn_seq(a, in ? b0 + lane : 0);
        const int rows = mine.nq * static_cast<int>(a.group.d);
        const int n = in && rows > a.few_rows ? (rows + m - 1) / m : 0;
        const int upto = before + wave_inclusive_sum(n, lane, a.batch - b0);
        const unsigned long long past = __ballot(upto > index);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            b = b0 + at;
            tile = __builtin_amdgcn_readlane(upto, at) - 1 - index;
            s = attn_pick(mine, at);
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// The work of a workgroup: a tile, and which of its spans of `span` keys.
__device__ __forceinline__ bool attn_find_work(const AttnArgs &a, int index, int m, int &b, int &tile, int &split,
                                               int &span, AttnSeq &s)
{
    split = blockIdx.y;
    span = a.tile_chunk;
    return attn_find_tile(a, index, m, b, tile, s);
}

// Trees: where even_parts says so, a sequence a lane, with spans of its own. All workgroups come to the same sizes.
__device__ __forceinline__ bool attn_find_work(const AttnTreeArgs &a, int index, int m, int &b, int &tile, int &split,
                                               int &span, AttnSeq &s)
{
    if (a.even_parts == 0) {
        return attn_find_work(static_cast<const AttnArgs &>(a), index, m, b, tile, split, span, s);
    }
    const int lane = threadIdx.x & 63;
    const AttnSeq mine = attn_seq(a, lane < a.batch ? lane : 0);
    const int rows = mine.nq * static_cast<int>(a.group.d);
    const int tiles = lane < a.batch && rows > a.few_rows ? (rows + m - 1) / m : 0;
    int keys = 0;
    if (tiles > 0) {
        const AttnKeys k = attn_tile_keys(a, mine, 0, m);
        keys = max(k.last - k.first, 0);
    }
    auto parts_of = [&](int most) { return min((keys - 1) / most + 1, a.even_parts); };
    // the smallest span, in 64 keys, that makes at most so many workgroups
    auto least = [&](int workgroups) {
        int lo = a.even_least >> 6, hi = a.even_most >> 6;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            const int n = wave_inclusive_sum(tiles * parts_of(mid << 6), lane, a.batch);
            if (__builtin_amdgcn_readlane(n, 63) * a.kv_heads <= workgroups) {
                hi = mid;
            } else {
                lo = mid + 1;
            }
        }
        return lo << 6;
    };
    const int one = least(a.even_round), two = least(2 * a.even_round);
    const int parts = parts_of(2 * two + kAttnEvenCost < one ? two : one);
    const int each = ((keys + parts - 1) / parts + 63) & ~63;
    const int items = tiles * attn_splits(0, keys, max(each, 64));
    const int upto = wave_inclusive_sum(items, lane, a.batch);
    const unsigned long long past = __ballot(upto > index);
    if (past == 0) {
        return false;
    }
    b = __builtin_ctzll(past);
    s = attn_pick(mine, b);
    span = max(__builtin_amdgcn_readlane(each, b), 64);
    const int n = __builtin_amdgcn_readlane(tiles, b);
    const int at = index - __builtin_amdgcn_readlane(upto - items, b);
    split = at / n;
    tile = n - 1 - (at - split * n);
    if (threadIdx.x == 0) {
        a.even_chunk[b] = span;  // the same from all of the sequence's workgroups
    }
    return true;
}

template <typename T, typename C, int DP, int NW, bool kFull, typename A>
__global__ __launch_bounds__(64 * NW, attn_tile_groups<A>(sizeof(C), DP)) void attn_tile_kernel(A a)
{
    constexpr bool kTree = std::is_same<A, AttnTreeArgs>::value;
    constexpr bool kQuant = std::is_same<C, int8_t>::value;
    // The second product's type: int8 values are whole numbers in f16, which costs less than bf16 and rounds
    // the probabilities less.
    typedef typename std::conditional<kQuant, _Float16, T>::type P;
    typedef typename Half8<T>::type half8;
    typedef typename Half8<P>::type prob8;
    constexpr int kGroups = DP / 32;                // blocks of 4 pieces along a row
    constexpr int kTileBytes = 64 * DP * 2;         // of K or V
    constexpr int kM = 32 * NW;
    __shared__ __attribute__((aligned(1024))) int8_t lds[4 * kTileBytes];  // K of even and odd tiles, V of both
    __shared__ __attribute__((aligned(16))) int s_kept[4][4];              // [tile % 4][16-key block]
    // int8: the keys' scales and the values' factors, [K, V][tile % 2], and the values' logarithms
    __shared__ __attribute__((aligned(16))) float s_scale[2][2][kQuant ? 64 : 4];
    __shared__ __attribute__((aligned(16))) float s_log[2][kQuant ? 64 : 4];

    // the key heads of a tile side by side: with 8 (or a multiple), a head's tiles are all on one XCD, whose L2
    // its keys then pass once for them
    const int index = static_cast<int>(blockIdx.x) / a.kv_heads;
    const int kvh = static_cast<int>(blockIdx.x) - index * a.kv_heads;
    int b, tile, split, span;
    AttnSeq s;
    if (!attn_find_work(a, index, kM, b, tile, split, span, s)) {
        return;
    }
    const int group = static_cast<int>(a.group.d);
    const AttnKeys keys = attn_tile_keys(a, s, tile, kM);
    const int splits = attn_splits(keys.first, keys.last, span);
    if (split >= splits) {
        return;
    }
    const int lo = keys.first + split * span, hi = min(keys.last, lo + span);

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int32_t *table = a.table + b * a.ld_table;
    const C *kbase = static_cast<const C *>(a.k), *vbase = static_cast<const C *>(a.v);

    // this lane's row, and the keys that it sees
    const int rows = s.nq * group;
    const int row = tile * kM + 32 * wave + col;
    const bool live = row < rows;
    uint32_t head_in_group;
    const int token = static_cast<int>(fast_div(live ? row : rows - 1, a.group, head_in_group));
    const int head = kvh * group + static_cast<int>(head_in_group);
    int row_lo, row_hi;
    attn_row_keys(a, s, token, row_lo, row_hi);
    // the keys that every row of the workgroup sees
    const int all_lo = keys.all_first, all_hi = keys.all_last;

    half8 q[DP / 16];
    const T *qp = static_cast<const T *>(a.q) + (s.first + token) * a.q_ts + head * a.q_hs;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        half8 x = {};
        if (16 * i < a.head_dim) {
            x = *reinterpret_cast<const half8 *>(qp + 16 * i + 8 * h);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = static_cast<T>(static_cast<float>(x[e]) * a.sign);
        }
        q[i] = x;
    }

    f32x16 o[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
        o[i] = 0.0f;
    }
    // Sums of 2^(s - ref) and 2^(s - ref) v. `ref`, in log2, follows the maximum of s (int8: of s and the logarithm
    // of the value's scale, value_scale) over the keys that the row sees only when that has grown by more
    // than 8: until then the probabilities stay below 256 and the sums as they are.
    float ref = -INFINITY, l = 0.0f;
    bool repair = false;  // values that are no numbers were taken out of tiles that not every row sees

    // loads: this lane's key of a tile is 16 x block + lane / 4
    constexpr int kBlocks = 4 / NW;  // 16-key blocks a wave loads
    const int piece = (lane & 3) ^ ((((lane >> 3) & 1) << 1) | ((lane >> 4) & 1));
    KeyRow k_next[kBlocks], v_next[kBlocks];
    PageAsked asked[kBlocks];
    auto ask = [&](int j0) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            asked[i] = attn_page_of(a, table, min(j0 + 16 * (wave * kBlocks + i) + (lane >> 2), hi - 1));
        }
    };
    auto resolve = [&](int j0) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            v_next[i] = k_next[i];
            k_next[i] = attn_key(a, asked[i], kvh);
            k_next[i].kept &= j0 + 16 * (wave * kBlocks + i) + (lane >> 2) < hi;
        }
    };
    auto note_kept = [&](int tile) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            const unsigned long long kept = __ballot(k_next[i].kept);
            if (lane == 0) {
                s_kept[tile & 3][wave * kBlocks + i] = kept == ~0ull;
            }
        }
    };
    // 16-bit rows go to LDS directly, `which` (0: K, 1: V) of an even or odd tile
    auto load = [&](const KeyRow (&from)[kBlocks], const C *source, int which, int tile) {
        const int8_t *zeros = reinterpret_cast<const int8_t *>(kAttnZeros);
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            int8_t *to = lds + (2 * which + (tile & 1)) * kTileBytes + (wave * kBlocks + i) * kGroups * 1024;
            const int8_t *p =
                (from[i].kept ? reinterpret_cast<const int8_t *>(source + from[i].at) : zeros) + 16 * piece;
#pragma unroll
            for (int c = 0; c < kGroups; ++c) {
                const bool in = kFull || 32 * c + 8 * piece < a.head_dim;
                dma_lds16(in ? p + 64 * c : zeros, to + c * 1024);
            }
        }
    };
    // int8 rows pass through registers, where they become 16-bit whole numbers
    constexpr int kRaw = kQuant ? (DP + 63) / 64 : 1;
    u32x4 raw[2][kBlocks][kRaw];
    float raw_scale[2][kBlocks];
    auto load_raw = [&](const KeyRow (&from)[kBlocks], const C *source, const float *scales, int which) {
        const C *zeros = reinterpret_cast<const C *>(kAttnZeros);
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            const C *p = (from[i].kept ? source + from[i].at : zeros) + 16 * (lane & 3);
#pragma unroll
            for (int c = 0; c < kRaw; ++c) {
                const bool in = (kFull && DP % 64 == 0) || 64 * c + 16 * (lane & 3) < a.head_dim;
                raw[which][i][c] = *reinterpret_cast<const u32x4 *>(in ? p + 64 * c : zeros);
            }
            const long long at = (static_cast<long long>(from[i].page) * a.kv_heads + kvh) * a.page.d +
                                 from[i].offset;
            raw_scale[which][i] = *(from[i].kept ? scales + at : reinterpret_cast<const float *>(kAttnZeros));
        }
    };
    auto store_raw = [&](auto half, int which, int tile) {
        typedef decltype(half) H;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            const int block = wave * kBlocks + i;
            int8_t *to = lds + (2 * which + (tile & 1)) * kTileBytes + block * kGroups * 1024 + (lane >> 2) * 64;
            const int f = (((lane >> 3) & 1) << 1) | ((lane >> 4) & 1);
#pragma unroll
            for (int c = 0; c < kRaw; ++c) {
                H x[2];
                int8_to_half(raw[which][i][c], x);
                const int place = 2 * c + ((lane >> 1) & 1);
                if (DP % 64 != 0 && place >= kGroups) {
                    continue;
                }
                int8_t *at = to + place * 1024;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    *reinterpret_cast<H *>(at + ((2 * (lane & 1) + e) ^ f) * 16) = x[e];
                }
            }
            const int key = 16 * block + (lane >> 2);
            if (which == 0) {
                if ((lane & 3) == 0) {
                    s_scale[0][tile & 1][key] = raw_scale[0][i];
                }
                continue;
            }
            uint32_t any = 0;
#pragma unroll
            for (int c = 0; c < kRaw; ++c) {
                any |= raw[1][i][c][0] | raw[1][i][c][1] | raw[1][i][c][2] | raw[1][i][c][3];
            }
            const unsigned long long rows = __ballot(any != 0);
            const ValueScale v = value_scale(raw_scale[1][i], ((rows >> (lane & ~3)) & 15) == 0);
            if ((lane & 3) == 0) {
                s_scale[1][tile & 1][key] = v.factor;
                s_log[tile & 1][key] = v.log;
            }
        }
    };

    // operand addresses within a stage
    const int fk = (((col >> 1) & 1) << 1) | ((col >> 2) & 1);
    const int k_at = (col >> 4) * kGroups * 1024 + (col & 15) * 64 + ((h ^ (fk & 1)) | (fk & 2)) * 16;
    const int vr = 4 * h + ((lane >> 2) & 3);
    const int fv = (((vr >> 1) & 1) << 1) | ((vr >> 2) & 1);
    const int v_at = 2 * kTileBytes + vr * 64 + (((((lane >> 4) & 1) << 1) | ((lane >> 1) & 1)) ^ fv) * 16 +
                     (lane & 1) * 8;

    // Bit r of seen[t]: whether this lane's row sees the key of its score r of half t of a tile. Which keys are
    // kept is looked up again: this is for tiles at the edges.
    auto see = [&](int j0, uint32_t (&seen)[2]) {
        const KeyRow kr = attn_key(a, table, kvh, j0 + lane, hi);
        const unsigned long long kept = __ballot(kr.kept);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            // keys [row_lo, row_hi) of the 32, those kept, and of them this half-wave's: 4 of every 8
            const int below = min(max(row_lo - j0 - 32 * t, 0), 32);
            const int upto = min(max(row_hi - j0 - 32 * t, 0), 32);
            uint32_t in = static_cast<uint32_t>(kept >> (32 * t));
            in &= static_cast<uint32_t>((1ull << upto) - 1) & ~static_cast<uint32_t>((1ull << below) - 1);
            if constexpr (kTree) {
                in &= attn_tree_bits(a, s, token, j0 + 32 * t);
            }
            in >>= 4 * h;
            seen[t] = (in & 0xfu) | ((in >> 4) & 0xf0u) | ((in >> 8) & 0xf00u) | ((in >> 12) & 0xf000u);
        }
    };
    auto scale_scores = [&](f32x16 (&st)[2], int parity) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x4 y = *reinterpret_cast<const f32x4 *>(&s_scale[0][parity][32 * t + 2 * r + 4 * h]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    st[t][r + c] *= y[c];
                }
            }
        }
    };
    auto max_of = [&](const f32x16 (&st)[2]) {
        float x = st[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                x = fmaxf(x, st[t][r]);
            }
        }
        return max_across_halves(x);
    };
    // int8: the largest of s + logarithm that this lane's row sees in a tile. Where every row sees all of the keys
    // and their scales lie within 2^4 of the first one's, the largest score and 2^4 times that scale bound it
    // from above by 8 at most, for which the terms have room below: prompts of 4096 at heads of 64 / 128 / 256
    // take 177 / 231 / 503 us so and, of one run, 184 / 232 / 541 with every key's own summand.
    auto value_top = [&](const f32x16 (&st)[2], int parity, bool mixed) {
        const float mine = s_log[parity][lane];
        const float most = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(
                                                         __builtin_bit_cast(int, mine))) + 4.0f;
        if (!mixed && __all(mine <= most && (mine >= most - 8.0f || mine == kValueLogLeast))) {
            return __builtin_fmaf(max_of(st), a.scale, most);
        }
        float x = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x4 y = *reinterpret_cast<const f32x4 *>(&s_log[parity][32 * t + 2 * r + 4 * h]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    // a score of -infinity beside an infinite logarithm is a NaN, which the maximum passes over
                    x = fmaxf(x, __builtin_fmaf(st[t][r + c], a.scale, y[c]));
                }
            }
        }
        return max_across_halves(x);
    };
    float top = 0.0f;   // of a tile's scores, masks left out (int8: value_top of the tile's own step)
    bool kept = false;  // whether all of its keys are on pages that are kept
    // One tile: its scores are in `st`; the next one's go to `after`, their products between the exponentials
    // of this one's (a wave issues in order, so that the two kinds have to alternate). `odd`: the tile's
    // number's lowest bit.
    auto step = [&](f32x16 (&st)[2], f32x16 (&after)[2], int j0, int n, auto odd) {
        constexpr int kOdd = decltype(odd)::value;
        const bool more = j0 + 64 < hi, more2 = j0 + 128 < hi;
        if (more2) {
            if constexpr (kQuant) {
                load_raw(k_next, kbase, a.scale_k, 0);
            } else {
                load(k_next, kbase, 0, kOdd);
            }
            note_kept(n + 2);
        }
        if (more) {
            if constexpr (kQuant) {
                load_raw(v_next, vbase, a.scale_v, 1);
            } else {
                load(v_next, vbase, 1, kOdd ^ 1);
            }
        }
        ask(j0 + 192);
        const bool mixed = !kept || j0 < all_lo || j0 + 64 > all_hi;
        if (mixed) {
            uint32_t seen[2];
            see(j0, seen);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    st[t][r] = (seen[t] >> r) & 1 ? st[t][r] : -INFINITY;
                }
            }
        }
        if constexpr (kQuant) {
            top = value_top(st, kOdd, mixed);
        } else if (mixed) {
            top = max_of(st);
        }

        // operands are read from LDS a group of four ahead of their products
        const int8_t *k_base = lds + (kOdd ^ 1) * kTileBytes, *v_base = lds + kOdd * kTileBytes;
        auto key = [&](int i, int t) {
            return *reinterpret_cast<const u32x4 *>(k_base + (k_at ^ (32 * (i & 1))) +
                                                    (2 * t * kGroups + (i >> 1)) * 1024);
        };
        auto value = [&](int i, int u) {
            const int8_t *at = v_base + v_at + (u * kGroups + i) * 1024;
            const u32x2 x0 = lds_read_column4(at), x1 = lds_read_column4(at + 512);
            return u32x4{x0[0], x0[1], x1[0], x1[1]};
        };
        u32x4 x[2][4];
        constexpr int kKeys = attn_tile_groups<A>(sizeof(C), DP) > 2 ? 2 : 4;
#pragma unroll
        for (int e = 0; e < kKeys; ++e) {
            x[0][e] = key(e >> 1, e & 1);
        }

        const i32x4 kept4 = *reinterpret_cast<const i32x4 *>(s_kept[(n + 1) & 3]);
        float want = kQuant ? top : top * a.scale;
        want = want - ref > 8.0f ? want : ref;
        const float base_s = want == -INFINITY ? 0.0f : want;
        float alpha;
        if constexpr (kQuant) {
            alpha = value_half_step(ref, base_s);
            l = l * alpha * alpha;
            alpha *= alpha;
            // infinite: a score, or the scale of a value that the row sees
            l = want == INFINITY ? __builtin_nanf("") : l;
        } else {
            alpha = __builtin_amdgcn_exp2f(ref - base_s);
            l *= alpha;
        }
        ref = want;
        if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                o[i] = o[i] * alpha;
            }
        }
        prob8 p[4];
        float sum[2] = {0.0f, 0.0f};
        after[0] = 0.0f;
        after[1] = 0.0f;
        constexpr int kProducts = DP / 8;
        auto each = [&](int k, auto f) {  // the scores of step k
#pragma unroll
            for (int c = 32 * k / kProducts; c < 32 * (k + 1) / kProducts; ++c) {
                f(c >> 4, c & 15);
            }
        };
        // int8: the values' scales, read a step ahead of their use
        constexpr int kScales = 2 * ((32 + kProducts - 1) / kProducts);
        float scales[kScales];
        auto read_scale = [&](int t, int r) {
            scales[(16 * t + r) % kScales] = s_scale[1][kOdd][32 * t + 8 * (r >> 2) + 4 * h + (r & 3)];
        };
        auto use = [&](int t, int r) {
            float e = st[t][r];
            sum[t] += e;
            if constexpr (kQuant) {
                e *= scales[(16 * t + r) % kScales];
            }
            prob8 &to = p[2 * t + (r >> 3)];
            to[r & 7] = static_cast<P>(e);
            if ((r & 7) == 7) {
                asm volatile("" : "+v"(to));
            }
        };
#pragma unroll
        for (int k = 0; k < kProducts; ++k) {
            if (k % kKeys == 0 && k + kKeys < kProducts) {
#pragma unroll
                for (int e = 0; e < kKeys; ++e) {
                    x[(k / kKeys + 1) & 1][e] = key((k + kKeys + e) >> 1, e & 1);
                }
            }
            after[k & 1] =
                mfma32(__builtin_bit_cast(half8, x[k / kKeys & 1][k % kKeys]), q[k >> 1], after[k & 1]);
            if constexpr (kQuant) {
                each(k, read_scale);
            }
            // exponentials of this step's scores, and what the last step's are for
            each(k, [&](int t, int r) {
                st[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][r], a.scale, -base_s));
            });
            if (k > 0) {
                each(k - 1, use);
                // holds them here: the compiler would sink all of it below the products
                asm volatile("" : "+v"(sum[0]), "+v"(sum[1]));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        each(kProducts - 1, use);
        l += sum[0] + sum[1];

        if constexpr (!kQuant) {
            if (mixed) {
                // values that are no numbers, which not every row may meet: all waves look at their share
                u32x4 *share = reinterpret_cast<u32x4 *>(lds + (2 + kOdd) * kTileBytes) + tid;
                bool bad = false;
#pragma unroll
                for (int i = 0; i < kTileBytes / 16; i += 64 * NW) {
                    const u32x4 y = share[i];
                    bad |= any_not_finite<T>(y[0]) || any_not_finite<T>(y[1]) || any_not_finite<T>(y[2]) ||
                           any_not_finite<T>(y[3]);
                }
                if (__syncthreads_or(bad)) {
                    for (int i = 0; i < kTileBytes / 16; i += 64 * NW) {
                        u32x4 clean, code;
                        split_not_finite<T>(share[i], clean, code);
                        share[i] = clean;
                    }
                    repair = true;
                    __syncthreads();
                }
            }
        }
        constexpr int kAhead = kGroups % 4 == 0 ? 4 : kGroups % 3 == 0 ? 3 : 2, kParts = 4 * kGroups / kAhead;
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            x[0][e] = value(e % kGroups, e / kGroups);
        }
        top = after[0][0];
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            if (k + 1 < kParts) {
#pragma unroll
                for (int e = 0; e < kAhead; ++e) {
                    const int at = (k + 1) * kAhead + e;
                    x[(k + 1) & 1][e] = value(at % kGroups, at / kGroups);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                const int at = k * kAhead + e;
                o[at % kGroups] =
                    mfma32(__builtin_bit_cast(prob8, x[k & 1][e]), p[at / kGroups], o[at % kGroups]);
                if constexpr (!kQuant) {
                    // the next tile's maximum, held between the products as the exponentials are
#pragma unroll
                    for (int c = 8 * at / kGroups; c < 8 * (at + 1) / kGroups; ++c) {
                        top = fmaxf(top, after[c >> 4][c & 15]);
                    }
                    asm volatile("" : "+v"(top));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        kept = __builtin_amdgcn_readfirstlane(kept4[0] & kept4[1] & kept4[2] & kept4[3]) != 0;
        if constexpr (kQuant) {
            scale_scores(after, kOdd ^ 1);
            if (more2) {
                store_raw(half8(), 0, kOdd);
            }
            if (more) {
                store_raw(prob8(), 1, kOdd ^ 1);
            }
        } else {
            top = max_across_halves(top);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        resolve(j0 + 192);
        __syncthreads();
    };

    if (lo < hi) {
        f32x16 even[2], odd[2];
        // K of tiles 0 and 1, V of tile 0
        ask(lo);
        resolve(lo);
        ask(lo + 64);
        resolve(lo + 64);
        note_kept(1);
        if constexpr (kQuant) {
            load_raw(k_next, kbase, a.scale_k, 0);
            store_raw(half8(), 0, 1);
            load_raw(v_next, kbase, a.scale_k, 0);
            load_raw(v_next, vbase, a.scale_v, 1);
            store_raw(half8(), 0, 0);
            store_raw(prob8(), 1, 0);
        } else {
            load(v_next, kbase, 0, 0);
            load(k_next, kbase, 0, 1);
            load(v_next, vbase, 1, 0);
        }
        ask(lo + 128);
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            const unsigned long long kept = __ballot(v_next[i].kept);
            if (lane == 0) {
                s_kept[0][wave * kBlocks + i] = kept == ~0ull;
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        resolve(lo + 128);
        __syncthreads();
        const i32x4 kept4 = *reinterpret_cast<const i32x4 *>(s_kept[0]);
        kept = __builtin_amdgcn_readfirstlane(kept4[0] & kept4[1] & kept4[2] & kept4[3]) != 0;
        even[0] = 0.0f;
        even[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const u32x4 k = *reinterpret_cast<const u32x4 *>(lds + (k_at ^ (32 * (i & 1))) +
                                                                 (2 * t * kGroups + (i >> 1)) * 1024);
                even[t] = mfma32(__builtin_bit_cast(half8, k), q[i], even[t]);
            }
        }
        if constexpr (kQuant) {
            scale_scores(even, 0);
        }
        top = max_of(even);
        __syncthreads();
        for (int j0 = lo, n = 0;;) {
            step(even, odd, j0, n, std::integral_constant<int, 0>());
            j0 += 64;
            if (j0 >= hi) {
                break;
            }
            step(odd, even, j0, n + 1, std::integral_constant<int, 1>());
            j0 += 64;
            n += 2;
            if (j0 >= hi) {
                break;
            }
        }
    }

    if constexpr (!kQuant) {
        if (repair) {
            // The tiles that not every row sees once more: what their values that are no numbers make of the rows
            // that do see them.
            for (int j0 = lo; j0 < hi; j0 += 64) {
                ask(j0);
                resolve(j0);
                load(k_next, vbase, 1, 0);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                bool all_kept = true;
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) {
                    all_kept &= k_next[i].kept;
                }
                if (__syncthreads_or(!all_kept) || j0 < all_lo || j0 + 64 > all_hi) {
                    uint32_t seen[2];
                    see(j0, seen);
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t bits = seen[u >> 1] >> (8 * (u & 1));
                        half8 see1;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            see1[e] = static_cast<T>((bits >> e) & 1 ? 1.0f : 0.0f);
                        }
#pragma unroll
                        for (int i = 0; i < DP / 32; ++i) {
                            const int8_t *at = lds + v_at + (u * kGroups + i) * 1024;
                            const u32x2 x0 = lds_read_column4(at), x1 = lds_read_column4(at + 512);
                            u32x4 clean, code;
                            split_not_finite<T>(u32x4{x0[0], x0[1], x1[0], x1[1]}, clean, code);
                            f32x16 count = 0.0f;
                            count = mfma32(__builtin_bit_cast(half8, code), see1, count);
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                o[i][r] += not_finite_term(count[r]);
                            }
                        }
                    }
                }
                __syncthreads();
            }
        }
    }

    if (!live) {
        return;
    }
    l += __shfl_xor(l, 32);
    const long long part = splits == 1 ? -1
                                       : attn_few_parts(a) +
                                             (static_cast<long long>(split) * a.q_tokens + s.first + token) *
                                                 a.q_heads +
                                             head;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            float out[4] = {o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
#pragma unroll
            for (int c = 0; kQuant && c < 4; ++c) {
                out[c] *= kValueUp;
            }
            attn_put<T, 4>(a, part, s.first + token, head, 32 * i + 2 * r + 4 * h, out, ref, l);
        }
    }
}

}  // namespace
}  // namespace tqt
