// Attention of few rows: sequences with at most 16 rows to a key head (one decoded token of up to 16 query
// heads, or a few tokens of fewer).
//
// Bound by the cache's bytes: per key 2 d elements are read once for 4 d 16 flops on the matrix cores. The
// batch's keys are cut into units of 128 for each key head, and the workgroups that fit the chip at once take
// equal runs of units, across sequences: 64 sequences of 2048 to 8192 keys (bf16, 8 key heads of 128) take
// 256-268 us (5.0-5.3 TB/s; reads alone reach 6.3), 307 with a workgroup for each sequence and key head,
// 335-357 with two to eight. A sequence that a run ends in leaves a part for attn_join.hpp.
//
// A workgroup is four independent waves; wave w takes the 32-key tiles w, w + 4, ... of its keys, with sums of
// its own, and the four meet once per sequence. No barrier in the loop. A tile's keys and values are in
// registers one tile ahead of their use (16 KB a wave in flight at d 128, 128 KB a CU), their pages another
// tile ahead: at three waves a SIMD instead of two the registers spill, and a reload from scratch waits for
// every load before it (797 instead of 351 us).
//
// With the keys as the rows of the first product, S^T = K Q^T, each lane holds 4 + 4 keys of one query: the
// softmax is 8 values in a lane and two exchanges, its statistics are one value a lane, and P^T is the second
// operand of O^T = V^T P^T as it stands. K comes from memory in the operand's layout; V goes through a wave's
// own LDS, which is read down its columns. Int8 rows become 16-bit whole numbers on the way (exactly), their
// scales go to the scores and the probabilities (32 sequences of 1024-4096 keys, 32 key heads of 128, f16: 150 us,
// 4.7 TB/s).
#pragma once

#include "attn_common.hpp"

namespace tqt {
namespace {

// DP: head_dim rounded up to 64, 128 or 256.
template <typename T, typename C, int DP>
struct FewRowTile
{
    static constexpr bool kQuant = std::is_same<C, int8_t>::value;
    static constexpr int kPieces = DP * static_cast<int>(sizeof(C)) / 64;  // 16-byte pieces of a row per lane
    static constexpr int kStride = DP * 2 + 16;                           // bytes of a value row in LDS
    static constexpr int kWaveBytes = 32 * kStride + (kQuant ? 384 : 0);
};

template <typename T, typename C, int DP, bool kFull>
__global__ __launch_bounds__(64 * kAttnFewRowWaves, DP == 256 ? 1 : 2) void attn_few_row_kernel(AttnArgs a)
{
    typedef FewRowTile<T, C, DP> Tile;
    typedef typename Half8<T>::type half8;
    constexpr bool kQuant = Tile::kQuant;
    // the second product's type: int8 values are whole numbers in f16
    typedef typename std::conditional<kQuant, _Float16, T>::type P;
    typedef typename Half8<P>::type prob8;
    constexpr int kPieces = Tile::kPieces, kSteps = DP / 32, kStride = Tile::kStride;
    constexpr int kElems = 16 / static_cast<int>(sizeof(C));  // elements of a piece
    __shared__ __attribute__((aligned(16))) char lds[kAttnFewRowWaves * Tile::kWaveBytes];
    __shared__ float s_m[kAttnFewRowWaves][16], s_l[kAttnFewRowWaves][16];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int col = lane & 15, g = lane >> 4;
    const int group = static_cast<int>(a.group.d);
    char *mine = lds + wave * Tile::kWaveBytes;
    const int wg = static_cast<int>(blockIdx.x);
    int total;
    FewRowBatch batch;
    const int run = few_row_run(a, lane, total, batch);
    int unit = wg * run;
    const int end = min(unit + run, total);

    // one sequence and key head after another, each as far as the run goes
    while (unit < end) {
        if (a.batch > 64) {
            int before = 0;
            for (int b0 = 0; b0 < a.batch; b0 += 64) {
                few_row_batch(a, b0, before, lane, batch);
                before = __shfl(batch.upto, 63);
                if (before > unit) {
                    break;
                }
            }
        }
        const int in_batch = __builtin_ctzll(__ballot(batch.upto > unit));
        const int b = batch.b0 + in_batch;
        AttnSeq s;
        FewRowWork work;
        few_row_pick(batch, in_batch, s, work);
        const int before = __builtin_amdgcn_readlane(batch.upto, in_batch) - work.units * a.kv_heads;
        const int rows = s.nq * group;
        const int in_seq = __builtin_amdgcn_readfirstlane(unit - before);
        const int kvh = in_seq / work.units, unit0 = in_seq - kvh * work.units;
        const int unit1 = min(work.units, unit0 + (end - unit));
        unit += unit1 - unit0;
        const int lo = work.first + unit0 * kAttnFewRowUnit;
        const int hi = unit1 == work.units ? work.last : lo + (unit1 - unit0) * kAttnFewRowUnit;
        const bool whole = unit1 - unit0 == work.units;
        const long long part = whole ? -1 : (2ll * wg + (unit0 == 0)) * kAttnFewRows;
        const int32_t *table = a.table + b * a.ld_table;
        const C *kbase = static_cast<const C *>(a.k), *vbase = static_cast<const C *>(a.v);
        // this lane's row, and the keys that it sees
        const bool live = col < rows;
        uint32_t head_in_group;
        const int token = static_cast<int>(fast_div(live ? col : 0, a.group, head_in_group));
        const int head = kvh * group + static_cast<int>(head_in_group);
        int row_lo, row_hi;
        attn_bounds(a, s, s.pos0 + token, row_lo, row_hi);
        if (!live) {
            row_hi = 0;
        }
        // keys outside [all_lo, all_hi) are not seen by every row
        int all_lo, all_hi, unused;
        attn_bounds(a, s, s.pos0, unused, all_hi);
        attn_bounds(a, s, s.pos0 + s.nq - 1, all_lo, unused);

        // Q^T: the elements that the pieces of K bring in the same steps
        half8 q[kSteps];
        const T *qp = static_cast<const T *>(a.q) + (s.first + token) * a.q_ts + head * a.q_hs;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int d0 = kQuant ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g;
            half8 x = {};
            if (live && d0 < a.head_dim) {
                x = *reinterpret_cast<const half8 *>(qp + d0);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = static_cast<T>(static_cast<float>(x[e]) * a.sign);
            }
            q[i] = x;
        }

        f32x4 o[DP / 16];
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            o[i] = 0.0f;
        }
        // sums of 2^(s - ref) and 2^(s - ref) v; `ref` (log2) is the maximum so far of s, for int8 of s and the
        // logarithm of the value's scale (value_scale), over the keys that the row sees
        float ref = -INFINITY, l = 0.0f;

        // a tile's rows: this lane's are keys col and 16 + col; their pages are asked for a tile ahead
        u32x4 kx[2][kPieces], vx[2][kPieces];
        float sk = 0.0f, sv = 0.0f;  // int8: the scales of key lane % 32
        PageAsked asked[2];
        bool kept[2];
        auto ask = [&](int j) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                asked[t] = attn_ask_page(a, table, j + 16 * t + col, hi);
            }
        };
        auto fetch = [&]() {
            const C *zeros = reinterpret_cast<const C *>(kAttnZeros);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const KeyRow r = attn_key(a, asked[t], kvh);
                kept[t] = r.kept;
                const C *kp = (r.kept ? kbase + r.at : zeros) + g * kElems;
                const C *vp = (r.kept ? vbase + r.at : zeros) + g * kElems;
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const int d0 = 4 * i * kElems;
                    const bool in = kFull || d0 + g * kElems < a.head_dim;
                    kx[t][i] = *reinterpret_cast<const u32x4 *>(in ? kp + d0 : zeros);
                    vx[t][i] = *reinterpret_cast<const u32x4 *>(in ? vp + d0 : zeros);
                }
                if constexpr (kQuant) {
                    if (t == ((lane >> 4) & 1)) {
                        const long long at =
                            (static_cast<long long>(r.kept ? r.page : 0) * a.kv_heads + kvh) * a.page.d + r.offset;
                        sk = r.kept ? a.scale_k[at] : 0.0f;
                        sv = r.kept ? a.scale_v[at] : 0.0f;
                    }
                }
            }
        };

        int j0 = lo + 32 * wave;
        if (j0 < hi) {
            ask(j0);
            fetch();
            ask(j0 + kAttnFewRowUnit);
        }
        for (; j0 < hi; j0 += kAttnFewRowUnit) {
            // S^T
            f32x4 st[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                st[t] = 0.0f;
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    if constexpr (kQuant) {
                        half8 h[2];
                        int8_to_half(kx[t][i], h);
                        st[t] = mfma16(h[0], q[2 * i], st[t]);
                        st[t] = mfma16(h[1], q[2 * i + 1], st[t]);
                    } else {
                        st[t] = mfma16(__builtin_bit_cast(half8, kx[t][i]), q[i], st[t]);
                    }
                }
            }
            // V into LDS
            wave_lds_fence();
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                char *row = mine + (16 * t + col) * kStride;
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    if constexpr (kQuant) {
                        prob8 h[2];
                        int8_to_half(vx[t][i], h);
                        *reinterpret_cast<prob8 *>(row + 128 * i + 32 * g) = h[0];
                        *reinterpret_cast<prob8 *>(row + 128 * i + 32 * g + 16) = h[1];
                    } else {
                        *reinterpret_cast<u32x4 *>(row + 64 * i + 16 * g) = vx[t][i];
                    }
                }
            }
            // int8: the keys' scales, the values' factors and logarithms
            float *scales = reinterpret_cast<float *>(mine + 32 * kStride);
            if constexpr (kQuant) {
                uint32_t any[2] = {0, 0};
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) {
                        any[t] |= vx[t][i][0] | vx[t][i][1] | vx[t][i][2] | vx[t][i][3];
                    }
                }
                // this lane's scale is that of key lane % 32, whose row lanes col, col + 16, ... have
                const unsigned long long rows0 = __ballot(any[0] != 0), rows1 = __ballot(any[1] != 0);
                const unsigned long long rows = (lane & 16) != 0 ? rows1 : rows0;
                const ValueScale v = value_scale(sv, ((rows >> col) & 0x0001000100010001ull) == 0);
                if (lane < 32) {
                    scales[lane] = sk;
                    scales[32 + lane] = v.factor;
                    scales[64 + lane] = v.log;
                }
            }
            const unsigned long long kept0 = __ballot(kept[0]), kept1 = __ballot(kept[1]);
            const uint32_t keptmask = static_cast<uint32_t>(kept0 & 0xffff) |
                                      (static_cast<uint32_t>(kept1 & 0xffff) << 16);
            const int jt = j0;
            bool bad = false;
            const bool mixed = jt < all_lo || jt + 32 > all_hi;
            if constexpr (!kQuant) {
                if (mixed) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                bad |= any_not_finite<T>(vx[t][i][e]);
                            }
                        }
                    }
                    bad = __any(bad);
                }
            }
            wave_lds_fence();
            if (j0 + kAttnFewRowUnit < hi) {
                fetch();
                ask(j0 + 2 * kAttnFewRowUnit);
            }

            // softmax of this lane's 8 keys: 16 t + 4 g + r
            float top = -INFINITY;
            uint32_t seen = 0, in = keptmask;
            {
                const int below = min(max(row_lo - jt, 0), 32), upto = min(max(row_hi - jt, 0), 32);
                in &= static_cast<uint32_t>((1ull << upto) - 1) & ~static_cast<uint32_t>((1ull << below) - 1);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x4 ks = 1.0f, log = 0.0f;
                if constexpr (kQuant) {
                    ks = *reinterpret_cast<f32x4 *>(scales + 16 * t + 4 * g);
                    log = *reinterpret_cast<f32x4 *>(scales + 64 + 16 * t + 4 * g);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = 16 * t + 4 * g + r;
                    const bool see = (in >> key) & 1;
                    seen |= static_cast<uint32_t>(see) << (4 * t + r);
                    float x = st[t][r];
                    if constexpr (kQuant) {
                        x *= ks[r];
                    }
                    st[t][r] = see ? x * a.scale : -INFINITY;
                    // a NaN stays one: exp2 of it, below (that of a score of -infinity beside an infinite
                    // logarithm is passed over)
                    top = fmaxf(top, kQuant ? st[t][r] + log[r] : st[t][r]);
                }
            }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            top = fmaxf(ref, top);
            const float base = top == -INFINITY ? 0.0f : top;
            float alpha;
            if constexpr (kQuant) {
                alpha = value_half_step(ref, base);
                l = l * alpha * alpha;
                alpha *= alpha;
                // infinite: a score, or the scale of a value that the row sees
                l = top == INFINITY ? __builtin_nanf("") : l;
            } else {
                alpha = __builtin_amdgcn_exp2f(ref - base);
                l *= alpha;
            }
            ref = top;
            prob8 p;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x4 vsc = 1.0f;
                if constexpr (kQuant) {
                    vsc = *reinterpret_cast<f32x4 *>(scales + 32 + 16 * t + 4 * g);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float e = __builtin_amdgcn_exp2f(st[t][r] - base);
                    l += e;
                    if constexpr (kQuant) {
                        e *= vsc[r];
                    }
                    p[4 * t + r] = static_cast<P>(e);
                }
            }
            const char *columns = mine + (4 * g + (col >> 2)) * kStride + 8 * (lane & 3);
            auto value = [&](int i) {
                const u32x2 x0 = lds_read_column4(columns + 32 * i);
                const u32x2 x1 = lds_read_column4(columns + 32 * i + 16 * kStride);
                return u32x4{x0[0], x0[1], x1[0], x1[1]};
            };
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                o[i] = o[i] * alpha;
            }
            if constexpr (!kQuant) {
                if (bad) {
                    half8 see1;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        see1[e] = static_cast<T>((seen >> e) & 1 ? 1.0f : 0.0f);
                    }
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i) {
                        u32x4 clean, code;
                        split_not_finite<T>(value(i), clean, code);
                        const f32x4 count =
                            mfma16(__builtin_bit_cast(half8, code), see1, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            o[i][r] += not_finite_term(count[r]);
                        }
                    }
                    wave_lds_fence();
                    for (int i = lane; i < 32 * DP / 8; i += 64) {
                        u32x4 *at = reinterpret_cast<u32x4 *>(mine + (i / (DP / 8)) * kStride + 16 * (i % (DP / 8)));
                        u32x4 clean, code;
                        split_not_finite<T>(*at, clean, code);
                        *at = clean;
                    }
                    wave_lds_fence();
                }
            }
            // O^T
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                o[i] = mfma16(__builtin_bit_cast(prob8, value(i)), p, o[i]);
            }
        }

        // the four waves meet: sums of the lanes of a row, then of the waves
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        wave_lds_fence();
        float *mo = reinterpret_cast<float *>(mine);  // [16][DP]
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            *reinterpret_cast<f32x4 *>(mo + col * DP + 16 * i + 4 * g) = kQuant ? o[i] * kValueUp : o[i];
        }
        if (lane < 16) {
            s_m[wave][lane] = ref;
            s_l[wave][lane] = l;
        }
        __syncthreads();
        constexpr int kThreads = 4 * kAttnFewRowWaves, kOut = DP / kThreads;  // threads along a row, elements of each
        const int r = tid / kThreads, d0 = (tid % kThreads) * kOut;
        if (r < rows) {
            float mm = s_m[0][r];
#pragma unroll
            for (int w = 1; w < kAttnFewRowWaves; ++w) {
                mm = fmaxf(mm, s_m[w][r]);
            }
            const float base = mm == -INFINITY ? 0.0f : mm;
            float sum = 0.0f, acc[kOut] = {};
#pragma unroll
            for (int w = 0; w < kAttnFewRowWaves; ++w) {
                float part = s_l[w][r];
                const float f = part_factor<kQuant>(s_m[w][r], base, part);
                sum += part;
                const float *from = reinterpret_cast<const float *>(lds + w * Tile::kWaveBytes) + r * DP + d0;
#pragma unroll
                for (int e = 0; e < kOut; ++e) {
                    acc[e] += from[e] * f;
                }
            }
            const int out_token = static_cast<int>(fast_div(r, a.group, head_in_group));
            attn_put<T, kOut>(a, part < 0 ? -1 : part + r, s.first + out_token,
                              kvh * group + static_cast<int>(head_in_group), d0, acc, mm, sum);
        }
        __syncthreads();
    }
}

}  // namespace
}  // namespace tqt
