// The rows of accepted tokens in a paged cache, moved behind the context, on gfx950.
//
// Bound by latency, and by the moved bytes where layers and sequences are many. One thread takes one 16-byte piece of
// a head's row through all of its sequence's moves, in their order: token base + keep[j] goes to base + j. As keep
// ascends, keep[j] >= j, so a row is read before anything is written to it, whoever is ahead: no other thread has
// this piece. Eight moves are loaded together, then stored: a later move's row lies past every place of an earlier
// one. List, lengths and table entries are the same for all threads of a sequence and come from the caches. One
// sequence, or 64 with 8 layers: 2.8-4.4 us, most of it the launch and four dependent loads (lengths, list, pages, rows);
// the call takes the host 6.5.
#include "fast_div.hpp"
#include "paged_kv.hpp"
#include "tqt_hip_common.hpp"
#include "tqt_kv_keep_gfx950.h"

#include <algorithm>
#include <type_traits>

namespace tqt {
namespace {

constexpr int kKeepThreads = 256;
constexpr int kKeepAtOnce = 8;

struct KeepArgs
{
    const int32_t *q_start, *kv_len, *keep, *keep_len, *table;
    const int64_t *slots;
    const int32_t *positions;
    int32_t *kv_len_out;
    long long ld_keep, ld_table;
    char *k, *v;
    float *scale_k, *scale_v;
    long long page_bytes, token_bytes, head_bytes, layer_bytes, scale_layer;
    int max_keep, num_pages, kv_heads, most_len, tokens;
    FastDiv page, pieces, heads, batch;
    uint32_t items;  // layers x batch x (k, v) x heads x pieces
};

// Where token j of a sequence is: its page (-1: none of the cache) and the offset in it.
struct KeepPlace
{
    int page;
    uint32_t offset;
};

__device__ __forceinline__ KeepPlace keep_place(const KeepArgs &a, const int32_t *table, int j)
{
    KeepPlace p;
    const int page = table[fast_div(static_cast<uint32_t>(j), a.page, p.offset)];
    p.page = page >= 0 && page < a.num_pages ? page : -1;
    return p;
}

// Whether a sequence whose q_len > 0 drafted rows begin at `first` was refused: its kv_len does not count them. Its
// positions say so: those of tokens that kv_len counts are below it. The slots do not always: a refused sequence has
// none, but a token whose page is no page of the cache has none either, so the first row decides whose token, if
// it is counted, has a page.
__device__ __forceinline__ bool keep_refused(const KeepArgs &a, const int32_t *table, int first, int q_len, int kv_len)
{
    if (a.positions == nullptr && a.slots == nullptr) {
        return false;
    }
    if (first < 0 || first >= a.tokens) {
        return true;
    }
    if (a.positions != nullptr) {
        return a.positions[first] >= kv_len;
    }
    const int base = min(max(kv_len, 0), a.most_len) - q_len;
    for (int i = 0; i < q_len && first + i < a.tokens; ++i) {
        if (a.slots[first + i] >= 0) {
            return false;
        }
        if (base < 0 || keep_place(a, table, base + i).page >= 0) {
            return true;
        }
    }
    return false;
}

template <bool kQuant>
__global__ __launch_bounds__(kKeepThreads) void keep_kernel(KeepArgs a)
{
    const uint32_t item = blockIdx.x * kKeepThreads + threadIdx.x;
    if (item >= a.items) {
        return;
    }
    uint32_t piece, head, ub;
    uint32_t rest = fast_div(item, a.pieces, piece);
    rest = fast_div(rest, a.heads, head);
    const bool value = rest & 1;
    const uint32_t layer = fast_div(rest >> 1, a.batch, ub);
    const int b = static_cast<int>(ub);
    const int first = a.q_start[b];
    int q_len = max(a.q_start[b + 1] - first, 0);
    const int32_t *keep = a.keep + b * a.ld_keep, *table = a.table + b * a.ld_table;
    // one that brought nothing keeps its length, as one without drafted tokens
    if (q_len > 0 && keep_refused(a, table, first, q_len, a.kv_len[b])) {
        q_len = 0;
    }
    const int base = min(max(a.kv_len[b], 0), a.most_len) - q_len;
    const int most = base < 0 ? 0 : min(max(a.keep_len[b], 0), a.max_keep);
    char *rows = (value ? a.v : a.k) + layer * a.layer_bytes + head * a.head_bytes + 16 * piece;
    float *scales = nullptr;
    if constexpr (kQuant) {
        scales = (value ? a.scale_v : a.scale_k) + layer * a.scale_layer;
    }
    int n = 0, last = -1;
    for (bool more = true; more && n < most;) {
        int from[kKeepAtOnce];
        int moves = 0;
#pragma unroll
        for (int i = 0; i < kKeepAtOnce; ++i) {
            from[i] = n + i < most ? keep[n + i] : -1;
        }
#pragma unroll
        for (int i = 0; i < kKeepAtOnce; ++i) {
            more = more && from[i] > last && from[i] < q_len;
            last = from[i];
            moves += more;
        }
        KeepPlace src[kKeepAtOnce], dst[kKeepAtOnce];
#pragma unroll
        for (int i = 0; i < kKeepAtOnce; ++i) {
            src[i] = dst[i] = {-1, 0};
            if (i < moves && from[i] != n + i) {
                src[i] = keep_place(a, table, base + from[i]);
                dst[i] = keep_place(a, table, base + n + i);
            }
        }
        u32x4 x[kKeepAtOnce];
        float y[kKeepAtOnce];
        const bool has_scale = kQuant && piece == 0;
#pragma unroll
        for (int i = 0; i < kKeepAtOnce; ++i) {
            if (src[i].page >= 0 && dst[i].page >= 0) {
                x[i] = *reinterpret_cast<const u32x4 *>(rows + src[i].page * a.page_bytes +
                                                        src[i].offset * a.token_bytes);
                if (has_scale) {
                    y[i] = scales[(static_cast<long long>(src[i].page) * a.kv_heads + head) * a.page.d +
                                  src[i].offset];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kKeepAtOnce; ++i) {
            if (src[i].page >= 0 && dst[i].page >= 0) {
                *reinterpret_cast<u32x4 *>(rows + dst[i].page * a.page_bytes + dst[i].offset * a.token_bytes) =
                    x[i];
                if (has_scale) {
                    scales[(static_cast<long long>(dst[i].page) * a.kv_heads + head) * a.page.d +
                           dst[i].offset] = y[i];
                }
            }
        }
        n += moves;
    }
    if (a.kv_len_out != nullptr && layer == 0 && !value && head == 0 && piece == 0) {
        a.kv_len_out[b] = base < 0 ? 0 : base + n;
    }
}

const char *keep_error(const tqt_kv_keep_params *p, size_t bytes, bool quant)
{
    if (p == nullptr) {
        return "params == NULL";
    }
    if (p->batch == 0 || p->layers == 0) {
        return nullptr;
    }
    if (const char *e = paged_kv_error(p->kv, bytes, quant)) {
        return e;
    }
    const size_t top = 1u << 31;
    if (p->batch >= (1u << 16) || p->layers >= (1u << 16) || p->max_keep >= top || p->ld_table >= top) {
        return "batch, layers, max_keep or ld_table too large";
    }
    if (p->max_keep > p->ld_keep) {
        return "max_keep > ld_keep";
    }
    if (p->batch * p->layers * 2 * p->kv.kv_heads * (p->kv.head_dim * bytes / 16) >= top) {
        return "batch * layers * kv_heads * head_dim too large";
    }
    if (p->layers > 1 && (p->layer_stride * bytes) % 16 != 0) {
        return "the layers are off the 16-byte grid";
    }
    if (p->q_start == nullptr || p->kv_len == nullptr || p->keep_len == nullptr ||
        (p->keep == nullptr && p->max_keep > 0) || (p->block_table == nullptr && p->ld_table > 0)) {
        return "q_start / kv_len / keep / keep_len / block_table == NULL";
    }
    if (p->kv_len_out != nullptr && p->kv_len_out < p->kv_len + p->batch && p->kv_len < p->kv_len_out + p->batch) {
        return "kv_len_out overlaps kv_len";
    }
    if ((p->slots != nullptr || p->positions != nullptr) && p->tokens >= top) {
        return "tokens too large";
    }
    return nullptr;
}

template <typename C>
bool run_keep(const tqt_kv_keep_params *p, hipStream_t stream, const char *where)
{
    constexpr bool kQuant = std::is_same<C, int8_t>::value;
    if (p == nullptr) {
        return false;
    }
    const char *error = keep_error(p, sizeof(C), kQuant);
    TQT_REQUIRE(error == nullptr, error);
    if (p->batch == 0 || p->layers == 0) {
        return false;
    }
    const tqt_paged_kv &c = p->kv;
    KeepArgs a = {};
    a.q_start = p->q_start;
    a.kv_len = p->kv_len;
    a.keep = p->keep;
    a.keep_len = p->keep_len;
    a.table = p->block_table;
    a.kv_len_out = p->kv_len_out;
    a.slots = p->slots;
    a.positions = p->positions;
    a.tokens = static_cast<int>(p->slots != nullptr || p->positions != nullptr ? p->tokens : 0);
    a.ld_keep = static_cast<long long>(p->ld_keep);
    a.ld_table = static_cast<long long>(p->ld_table);
    a.k = static_cast<char *>(c.k);
    a.v = static_cast<char *>(c.v);
    a.scale_k = c.scale_k;
    a.scale_v = c.scale_v;
    a.page_bytes = static_cast<long long>(c.page_stride * sizeof(C));
    a.token_bytes = static_cast<long long>(c.token_stride * sizeof(C));
    a.head_bytes = static_cast<long long>(c.head_stride * sizeof(C));
    a.layer_bytes = static_cast<long long>(p->layer_stride * sizeof(C));
    a.scale_layer = static_cast<long long>(p->scale_layer_stride);
    a.max_keep = static_cast<int>(p->max_keep);
    a.num_pages = static_cast<int>(c.num_pages);
    a.kv_heads = static_cast<int>(c.kv_heads);
    a.most_len = static_cast<int>(std::min<size_t>(p->ld_table * c.page_size, (1u << 31) - 1));
    const size_t pieces = c.head_dim * sizeof(C) / 16;
    a.page = make_fast_div(static_cast<uint32_t>(c.page_size));
    a.pieces = make_fast_div(static_cast<uint32_t>(pieces));
    a.heads = make_fast_div(static_cast<uint32_t>(c.kv_heads));
    a.batch = make_fast_div(static_cast<uint32_t>(p->batch));
    a.items = static_cast<uint32_t>(p->layers * p->batch * 2 * c.kv_heads * pieces);
    hipLaunchKernelGGL((keep_kernel<kQuant>), dim3((a.items + kKeepThreads - 1) / kKeepThreads), dim3(kKeepThreads),
                       0, stream, a);
    check_launch(where);
    return true;
}

}  // namespace
}  // namespace tqt

using namespace tqt;

extern "C" {

#define TQT_KEEP_ENTRIES(NAME, C)                                                                     \
    const char *tqt_get_error_kv_keep_##NAME##_gfx950(const struct tqt_kv_keep_params *params)        \
    {                                                                                                 \
        return keep_error(params, sizeof(C), std::is_same<C, int8_t>::value);                         \
    }                                                                                                 \
    void tqt_run_kv_keep_##NAME##_gfx950_async(const struct tqt_kv_keep_params *params, void *stream) \
    {                                                                                                 \
        run_keep<C>(params, as_stream(stream), "tqt_run_kv_keep_" #NAME "_gfx950");                   \
    }                                                                                                 \
    void tqt_run_kv_keep_##NAME##_gfx950(const struct tqt_kv_keep_params *params)                     \
    {                                                                                                 \
        if (run_keep<C>(params, nullptr, "tqt_run_kv_keep_" #NAME "_gfx950")) {                       \
            finish_sync(nullptr, "tqt_run_kv_keep_" #NAME "_gfx950");                                 \
        }                                                                                             \
    }

TQT_KEEP_ENTRIES(f16, _Float16)
TQT_KEEP_ENTRIES(bf16, __bf16)
TQT_KEEP_ENTRIES(qsi8dx, int8_t)

}  // extern "C"
