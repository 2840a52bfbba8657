// Host side of the operators on packed documents (include/svl_hip.h): plans
// (lengths, masks and work items of a batch, in HBM) and the calls' checks.
// The reference has no counterpart of these operators; its one-axis rotation
// is src/tensor/kernels.rs:1014-1035 and its attention kernels.rs:1037-1135.
#include <climits>
#include <memory>
#include <new>
#include <numeric>

#include "host_common.hpp"
#include "packed.hpp"

using namespace svl;

namespace {

// The plan's device for the length of a call, the caller's again afterwards.
struct OnDevice {
    int before = -1;
    hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
    OnDevice(const OnDevice &) = delete;
};

template <class T>
svl_status upload(const std::vector<T> &v, T **d) {
    if (v.empty()) return SVL_OK;
    T *p = nullptr;
    HIP_TRY(hipMalloc((void **)&p, v.size() * sizeof(T)));
    *d = p;
    HIP_TRY(hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice));
    return SVL_OK;
}

// Makes a plan: build(plan) checks and lays it out on the host, bring(plan)
// takes it to the context's device. On failure nothing stays and *out is null.
template <class P, class Build, class Bring>
svl_status make_plan(svl_ctx *ctx, P **out, Build &&build, Bring &&bring) {
    if (!out) return fail(SVL_USAGE, "out is null");
    *out = nullptr;
    if (!ctx) return fail(SVL_USAGE, "context is null");
    try {
        auto plan = std::make_unique<P>();
        plan->device = ctx->device;
        ST_TRY(build(*plan));
        OnDevice on(ctx->device);  // ends after a failed plan has been freed
        HIP_TRY(on.err);
        const svl_status st = bring(*plan);
        if (st != SVL_OK) {
            plan.reset();
            return st;
        }
        *out = plan.release();
        return SVL_OK;
    } catch (const std::bad_alloc &) {
        return fail(SVL_LIMIT, "the plan does not fit in memory");
    }
}

bool aligned(const void *p, int64_t bytes) { return (uintptr_t)p % (uintptr_t)bytes == 0; }

// Rows and tokens: a tile past the last one still has 32-bit indexes. Workgroups:
// a launch counts its threads in 32 bits.
constexpr int64_t MAX_ROWS = INT32_MAX - 4095, MAX_WORKGROUPS = (INT64_C(1) << 23) - 1;
// Largest strides in elements: a row's offset then stays below 2^57 bytes, and
// a tile of 64 rows within 31 bits.
constexpr int64_t MAX_TOKEN_STRIDE = INT64_C(1) << 22, MAX_HEAD_STRIDE = INT64_C(1) << 40;

svl_status check_strides(int64_t token, int64_t head) {
    if (token < 0 || head < 0) return fail(SVL_USAGE, "a stride is negative");
    if (token > MAX_TOKEN_STRIDE)
        return fail(SVL_LIMIT, "a token stride of %lld elements is above 2^22", (long long)token);
    if (head > MAX_HEAD_STRIDE)
        return fail(SVL_LIMIT, "a head stride of %lld elements is above 2^40", (long long)head);
    return SVL_OK;
}

// Rows that are written do not share memory: the heads of a token lie within
// its stride, or the tokens of a head within the head's.
bool rows_apart(int64_t tokens, int64_t heads, int64_t token, int64_t head, int64_t hd) {
    if (tokens > 1 && token < hd) return false;
    if (heads > 1 && head < hd) return false;
    return tokens <= 1 || heads <= 1 || token >= (heads - 1) * head + hd ||
           head >= (tokens - 1) * token + hd;
}

}  // namespace

struct svl_position_plan {
    int device = 0;
    int64_t tokens = 0;
    PositionSegment *seg = nullptr;
    int32_t *block_seg = nullptr;
    ~svl_position_plan() {
        if (seg) (void)hipFree(seg);
        if (block_seg) (void)hipFree(block_seg);
    }
};

struct svl_attention_plan {
    int device = 0;
    svl_attention_shape shape{};
    MaskedShape tiles{};
    int64_t workspace = 0, planes_at = 0;  // bytes; planes behind the partial results
    int64_t q_rows = 0, kv_rows = 0;  // rows up to the last document's end
    int32_t n_work = 0, n_join = 0, join_vectors = 0, join_parts = 0, n_tiles = 0;
    AttnWork *work = nullptr;
    AttnJoin *join = nullptr;
    AttnTiles *key_tiles = nullptr;
    ~svl_attention_plan() {
        if (work) (void)hipFree(work);
        if (join) (void)hipFree(join);
        if (key_tiles) (void)hipFree(key_tiles);
    }
};

namespace {

svl_status fill_positions(svl_position_plan &plan, const svl_segment *segments, int64_t n,
                          std::vector<PositionSegment> &seg, std::vector<int32_t> &block_seg) {
    int64_t tokens = 0, at = 0;
    for (int64_t i = 0; i < n; ++i) {
        const svl_segment &s = segments[i];
        if (i > 0 && s.document < segments[i - 1].document)
            return fail(SVL_USAGE, "segment %lld: document %lld after document %lld", (long long)i,
                        (long long)s.document, (long long)segments[i - 1].document);
        if (i == 0 || s.document != segments[i - 1].document) at = 0;
        const bool grid = s.kind == SVL_SEGMENT_GRID;
        if (!grid && s.kind != SVL_SEGMENT_TEXT)
            return fail(SVL_USAGE, "segment %lld: kind %d is neither text nor grid", (long long)i,
                        s.kind);
        if (s.frames < 0 || (grid && (s.rows < 0 || s.cols < 0)))
            return fail(SVL_USAGE, "segment %lld has a negative size", (long long)i);
        if (grid && s.step < 1)
            return fail(SVL_USAGE, "segment %lld: step %d is below 1", (long long)i, s.step);
        int64_t count = s.frames, extent = s.frames;
        if (grid) {
            const int64_t area = (int64_t)s.rows * s.cols;
            if (area > 0 && s.frames > INT32_MAX / area)
                return fail(SVL_LIMIT, "segment %lld: more than 2^31 - 1 tokens", (long long)i);
            count = area * s.frames;
            extent = std::max<int64_t>((int64_t)s.step * (s.frames - 1) + 1,
                                       std::max(s.rows, s.cols));
        }
        if (count == 0) continue;
        if (at + extent > INT32_MAX)
            return fail(SVL_LIMIT, "segment %lld: a position reaches 2^31", (long long)i);
        if (tokens + count > MAX_ROWS) return fail(SVL_LIMIT, "more than 2^31 - 4096 tokens");
        PositionSegment d{(int32_t)tokens, (int32_t)at, 0, 1, 0};
        if (grid) {
            d.area = s.rows * s.cols;
            d.cols = s.cols;
            d.step = s.step;
        }
        seg.push_back(d);
        tokens += count;
        at += extent;
        while ((int64_t)block_seg.size() * POSITION_BLOCK < tokens)
            block_seg.push_back((int32_t)seg.size() - 1);
    }
    block_seg.push_back((int32_t)seg.size() - 1);
    plan.tokens = tokens;
    return SVL_OK;
}

// The order of launch. Workgroup b runs on XCD b % 8, and the groups of one
// document and KV head (beside each other in `work`) share their keys in its L2:
// whole ones go to the XCD with the least work, longest first, large ones in
// pieces of half an XCD's share. A piece takes its groups at a stride of the
// golden ratio, so that each has the short and the long ones of a causal mask;
// an XCD whose groups are all long would run a second round for a few of them
// (64 documents of 64-512 tokens: contiguous eighths 191 us, this order
// 161). Within an XCD the longest go first, and the short ones end the
// launch.
void order_work(std::vector<AttnWork> &work) {
    constexpr size_t XCDS = 8;
    auto cost = [](const AttnWork &w) { return (int64_t)(w.t1 - w.t0) + 2; };  // 2: start and end
    auto longer = [&](const AttnWork &a, const AttnWork &b) { return cost(a) > cost(b); };
    int64_t total = 0;
    for (const AttnWork &w : work) total += cost(w);
    struct Piece {
        std::vector<AttnWork> work;
        int64_t cost = 0;
    };
    std::vector<Piece> pieces;
    for (size_t i = 0; i < work.size();) {
        size_t n = 1;
        while (i + n < work.size() && work[i + n].q_row == work[i].q_row &&
               work[i + n].kvh == work[i].kvh)
            ++n;
        size_t stride = std::max<size_t>((size_t)((double)n * 0.618), 1);
        while (std::gcd(stride, n) > 1) ++stride;
        pieces.emplace_back();
        for (size_t k = 0; k < n; ++k) {
            if (pieces.back().cost * 2 * (int64_t)XCDS >= total) pieces.emplace_back();
            const AttnWork &w = work[i + k * stride % n];
            pieces.back().work.push_back(w);
            pieces.back().cost += cost(w);
        }
        i += n;
    }
    std::stable_sort(pieces.begin(), pieces.end(),
                     [](const Piece &a, const Piece &b) { return a.cost > b.cost; });
    Piece part[XCDS];
    for (Piece &p : pieces) {
        Piece *least = std::min_element(part, part + XCDS, [](const Piece &a, const Piece &b) {
            return a.cost < b.cost;
        });
        least->work.insert(least->work.end(), p.work.begin(), p.work.end());
        least->cost += p.cost;
    }
    size_t longest = 0;
    for (Piece &p : part) {
        std::stable_sort(p.work.begin(), p.work.end(), longer);
        longest = std::max(longest, p.work.size());
    }
    work.clear();
    for (size_t i = 0; i < longest; ++i)
        for (const Piece &p : part)
            if (i < p.work.size()) work.push_back(p.work[i]);
}

svl_status fill_attention(svl_attention_plan &plan, const int64_t *qo, const int64_t *ko,
                          const int64_t *prefix, int32_t documents, std::vector<AttnWork> &work,
                          std::vector<AttnJoin> &join, std::vector<AttnTiles> &tiles) {
    const svl_attention_shape &sh = plan.shape;
    const int64_t G = sh.num_heads / sh.num_kv_heads;
    int64_t most = 0;
    for (int32_t d = 0; d < documents; ++d) most = std::max(most, (qo[d + 1] - qo[d]) * G);
    plan.tiles = masked_shape(sh.dtype == SVL_BF16, (int)sh.head_dim, most);
    const int64_t KT = plan.tiles.keys, BV = plan.tiles.vectors;
    int64_t groups = 0, key_tiles = 0;
    for (int32_t d = 0; d < documents; ++d) {
        const int64_t ql = qo[d + 1] - qo[d];
        groups += (ql * G + BV - 1) / BV * sh.num_kv_heads;
        if (ql > 0) key_tiles += (ko[d + 1] - ko[d] + KT - 1) / KT * sh.num_kv_heads;
        if (groups > MAX_WORKGROUPS || (plan.tiles.planes > 0 && key_tiles > MAX_WORKGROUPS))
            return fail(SVL_LIMIT, "more than 2^23 - 1 groups of queries or tiles of keys");
    }
    int64_t total = 0;  // key tiles of all groups
    for (int32_t d = 0; d < documents; ++d) {
        const int64_t ql = qo[d + 1] - qo[d], kl = ko[d + 1] - ko[d];
        const int64_t pre = prefix ? std::min(prefix[d], kl) : 0;
        const int64_t shift = kl - ql;
        // laid out tiles: those that the document's queries see, from the first of them
        // (a window over a long cache) or of the prefix
        int64_t from = 0, to = 0;
        if (plan.tiles.planes > 0 && ql > 0) {
            int64_t lo = 0, hi = kl - 1;
            if (sh.causal) hi = std::min(hi, shift + ql - 1);
            if (sh.window >= 0) {
                lo = std::max(lo, shift - sh.window);
                hi = std::min(hi, shift + ql - 1 + sh.window);
            }
            to = (pre + KT - 1) / KT;
            if (hi >= lo) {
                from = to > 0 ? 0 : lo / KT;
                to = std::max(to, hi / KT + 1);
            }
        }
        const int64_t tile0 = (int64_t)tiles.size() - from;
        for (int64_t g = 0; g < sh.num_kv_heads; ++g)
            for (int64_t t = from; t < to; ++t)
                tiles.push_back({(int32_t)(ko[d] + t * KT), (int32_t)std::min(KT, kl - t * KT), (int32_t)g});
        for (int64_t g = 0; g < sh.num_kv_heads; ++g)
            for (int64_t v0 = 0; v0 < ql * G; v0 += BV) {
                // keys that some query of the group sees: the prefix and [lo, hi]
                const int64_t p_lo = v0 / G + shift,
                              p_hi = (std::min(v0 + BV, ql * G) - 1) / G + shift;
                int64_t lo = 0, hi = kl - 1;
                if (sh.causal) hi = std::min(hi, p_hi);
                if (sh.window >= 0) {
                    lo = std::max(lo, p_lo - sh.window);
                    hi = std::min(hi, p_hi + sh.window);
                }
                const int64_t pre_tiles = (pre + KT - 1) / KT;
                const int64_t first = std::max(lo / KT, pre_tiles);
                const int64_t seen =
                    pre_tiles + (hi >= lo ? std::max<int64_t>(hi / KT + 1 - first, 0) : 0);
                total += seen;
                // (keys past the last tile are never asked for, so main_key may pass them)
                work.push_back({(int32_t)qo[d], (int32_t)ql, (int32_t)ko[d], (int32_t)kl,
                                (int32_t)g, (int32_t)v0, (int32_t)pre, (int32_t)pre_tiles,
                                (int32_t)std::min<int64_t>(first * KT, INT32_MAX), 0,
                                (int32_t)seen, -1, (int32_t)(tile0 + g * (to - from))});
            }
    }
    // Groups that leave slots empty, or that are longer than half again the share of
    // one, are split over workgroups, whose parts a second launch joins.
    // Where a slot's share would be a few tiles, as much as a workgroup takes to
    // start, one round of two workgroups a CU does better than more, shorter ones
    // (single queries of 8 heads of 128 over 16 x 3000-9000 keys: 19.6 us against
    // 23.0; over 64 x 2000-8192 keys 46.9 against 40.8).
    // Nor does one group gain from a thousand parts (60000 keys: 16.8 us against 22.4).
    int64_t slots = plan.tiles.slots;
    if (total < 8 * 512 && (total > slots || work.size() < 16)) slots = std::min<int64_t>(slots, 512);
    if (plan.tiles.dim > 0 && 4 * (int64_t)work.size() < 3 * slots) {
        const int64_t each = std::max<int64_t>((total + slots - 1) / slots, plan.tiles.least);
        std::vector<AttnWork> split;
        int64_t used = 0;
        for (const AttnWork &w : work) {
            const int64_t parts = 2 * w.t1 > 3 * each ? (w.t1 + each - 1) / each : 1;
            if (parts > 1) {
                join.push_back({w.q_row, w.q_len, w.kvh, w.v0, (int32_t)used, (int32_t)parts});
                plan.join_parts = std::max(plan.join_parts, (int32_t)parts);
            }
            for (int64_t i = 0; i < parts; ++i) {
                AttnWork x = w;
                x.t0 = (int32_t)(w.t1 * i / parts);
                x.t1 = (int32_t)(w.t1 * (i + 1) / parts);
                x.slot = parts > 1 ? (int32_t)(used + i) : -1;
                split.push_back(x);
            }
            if (parts > 1) used += parts;
        }
        work.swap(split);
        plan.planes_at = used * masked_slot((int)BV, plan.tiles.dim) * (int64_t)sizeof(float);
    }
    order_work(work);
    plan.n_work = (int32_t)work.size();
    plan.n_tiles = (int32_t)tiles.size();
    plan.planes_at = (plan.planes_at + 15) / 16 * 16;
    plan.workspace = plan.planes_at + plan.n_tiles * masked_tile_bytes(plan.tiles);
    plan.n_join = (int32_t)join.size();
    plan.join_vectors = (int32_t)std::min(most, BV);
    plan.q_rows = qo[documents];
    plan.kv_rows = ko[documents];
    return SVL_OK;
}

svl_status check_offsets(const int64_t *off, int32_t documents, const char *what) {
    if (off[0] < 0) return fail(SVL_USAGE, "%s offsets start below 0", what);
    for (int32_t d = 0; d < documents; ++d)
        if (off[d + 1] < off[d])
            return fail(SVL_USAGE, "%s offset %d decreases", what, d + 1);
    if (off[documents] > MAX_ROWS) return fail(SVL_LIMIT, "more than 2^31 - 4096 %s rows", what);
    return SVL_OK;
}

}  // namespace

extern "C" {

svl_status svl_position_plan_create(svl_ctx *ctx, const svl_segment *segments, int64_t n,
                                    svl_position_plan **out) {
    std::vector<PositionSegment> seg;
    std::vector<int32_t> block_seg;
    return make_plan(
        ctx, out,
        [&](svl_position_plan &plan) {
            if (n < 0) return fail(SVL_USAGE, "segment count is negative");
            if (n > 0 && !segments) return fail(SVL_USAGE, "segments are null");
            return fill_positions(plan, segments, n, seg, block_seg);
        },
        [&](svl_position_plan &plan) {
            ST_TRY(upload(seg, &plan.seg));
            return upload(block_seg, &plan.block_seg);
        });
}

svl_status svl_position_plan_destroy(svl_position_plan *plan) {
    if (!plan) return SVL_OK;
    OnDevice on(plan->device);
    delete plan;
    return SVL_OK;
}

int64_t svl_position_plan_tokens(const svl_position_plan *plan) { return plan ? plan->tokens : 0; }

svl_status svl_axis_positions(const svl_position_plan *plan, int32_t *d_positions, void *stream) {
    if (!plan) return fail(SVL_USAGE, "plan is null");
    if (plan->tokens == 0) return SVL_OK;
    if (!d_positions) return fail(SVL_USAGE, "positions are null");
    if (!aligned(d_positions, 4)) return fail(SVL_USAGE, "positions are not aligned to 4 bytes");
    OnDevice on(plan->device);
    HIP_TRY(on.err);
    HIP_TRY(launch_axis_positions(plan->seg, plan->block_seg, plan->tokens, d_positions,
                                  (hipStream_t)stream));
    return SVL_OK;
}

svl_status svl_rope_axes(const svl_rope_rows *tensors, int32_t n_tensors, int32_t dtype,
                         const int32_t *d_positions, int64_t tokens, int32_t axes,
                         int64_t head_dim, const float *inv_freq, const uint8_t *pair_axis,
                         int64_t pairs, int32_t layout, void *stream) {
    if (!tensors || n_tensors < 1 || n_tensors > 2)
        return fail(SVL_USAGE, "rotation takes one or two tensors");
    if (dtype != SVL_F32 && dtype != SVL_BF16)
        return fail(SVL_UNSUPPORTED, "rotation of type %d: F32 and BF16 are supported", dtype);
    if (axes < 1 || axes > 4) return fail(SVL_USAGE, "%d axes are outside 1..=4", axes);
    if (layout != SVL_ROPE_HALF && layout != SVL_ROPE_ADJACENT && layout != SVL_ROPE_AXIAL)
        return fail(SVL_USAGE, "rotation layout %d is not known", layout);
    if (head_dim < 1 || head_dim > 1024)
        return fail(SVL_UNSUPPORTED, "head dim %lld is outside 1..=1024", (long long)head_dim);
    if (pairs < 0 || 2 * pairs > head_dim)
        return fail(SVL_USAGE, "%lld pairs do not fit head dim %lld", (long long)pairs,
                    (long long)head_dim);
    if (pairs > ROPE_MAX_PAIRS)
        return fail(SVL_UNSUPPORTED, "%lld pairs: at most %d are rotated", (long long)pairs,
                    ROPE_MAX_PAIRS);
    if (pairs > 0 && (!inv_freq || !pair_axis))
        return fail(SVL_USAGE, "frequencies or axes of the pairs are null");
    if (tokens < 0) return fail(SVL_USAGE, "token count is negative");
    if (tokens > MAX_ROWS) return fail(SVL_LIMIT, "more than 2^31 - 4096 tokens");
    RopeAxesArgs a{};
    a.pos = d_positions;
    a.tokens = tokens;
    a.axes = axes;
    a.hd = (int32_t)head_dim;
    a.pairs = (int32_t)pairs;
    const bool adjacent = layout == SVL_ROPE_ADJACENT;
    const int64_t size = dtype == SVL_BF16 ? 2 : 4, chunk = 16 / size;
    bool runs = pairs % chunk == 0, rows = head_dim % chunk == 0;  // in whole chunks
    for (int64_t j = 0, run = 0; j < pairs; ++j) {
        if (pair_axis[j] >= axes)
            return fail(SVL_USAGE, "pair %lld: axis %d of %d", (long long)j, pair_axis[j], axes);
        if (!std::isfinite(inv_freq[j]))
            return fail(SVL_USAGE, "pair %lld: frequency is not finite", (long long)j);
        a.inv_freq[j] = inv_freq[j];
        a.axis[j] = pair_axis[j];
        if (adjacent) {
            a.col[j] = (uint16_t)(2 * j);
            a.partner[j] = (uint16_t)(2 * j + 1);
        } else if (layout == SVL_ROPE_HALF) {
            a.col[j] = (uint16_t)j;
            a.partner[j] = (uint16_t)(j + pairs);
        } else {
            if (j > 0 && pair_axis[j] != pair_axis[j - 1]) run = j;
            int64_t end = j;
            while (end < pairs && pair_axis[end] == pair_axis[j]) ++end;
            a.col[j] = (uint16_t)(run + j);
            a.partner[j] = (uint16_t)(end + j);
            runs = runs && (end - run) % chunk == 0;
        }
    }
    bool copies = false;
    for (int i = 0; i < n_tensors; ++i) {
        const svl_rope_rows &r = tensors[i];
        if (r.heads < 0) return fail(SVL_USAGE, "head count is negative");
        if (r.heads > 32767) return fail(SVL_LIMIT, "more than 32767 heads");
        if (r.heads == 0 || tokens == 0) continue;
        if (!r.in || !r.out) return fail(SVL_USAGE, "rows are null");
        ST_TRY(check_strides(r.in_token_stride, r.in_head_stride));
        ST_TRY(check_strides(r.out_token_stride, r.out_head_stride));
        if (!rows_apart(tokens, r.heads, r.out_token_stride, r.out_head_stride, head_dim))
            return fail(SVL_USAGE, "output rows overlap");
        if (r.in == r.out && ((r.heads > 1 && r.in_head_stride != r.out_head_stride) ||
                              (tokens > 1 && r.in_token_stride != r.out_token_stride)))
            return fail(SVL_USAGE, "rows rotated in place have two strides");
        if (!aligned(r.in, size) || !aligned(r.out, size))
            return fail(SVL_USAGE, "rows are not aligned to their type");
        a.in[i] = r.in;
        a.out[i] = r.out;
        a.heads[i] = (int32_t)r.heads;
        a.in_tok[i] = r.in_token_stride;
        a.in_head[i] = r.in_head_stride;
        a.out_tok[i] = r.out_token_stride;
        a.out_head[i] = r.out_head_stride;
        for (int64_t st : {r.heads > 1 ? r.in_head_stride : 0, r.heads > 1 ? r.out_head_stride : 0,
                           tokens > 1 ? r.in_token_stride : 0, tokens > 1 ? r.out_token_stride : 0})
            rows = rows && st % chunk == 0;
        rows = rows && aligned(r.in, 16) && aligned(r.out, 16);
        copies = copies || r.in != r.out;
    }
    if (copies) a.copied = (int32_t)(head_dim - 2 * pairs);
    if (tokens == 0 || a.heads[0] + a.heads[1] == 0 || (pairs == 0 && a.copied == 0)) return SVL_OK;
    if (pairs > 0 && !d_positions) return fail(SVL_USAGE, "positions are null");
    if (!aligned(d_positions, 4)) return fail(SVL_USAGE, "positions are not aligned to 4 bytes");
    const RopeForm form = !rows ? ROPE_SINGLE : runs ? ROPE_CHUNKS : ROPE_ROWS;
    HIP_TRY(launch_rope_axes(a, dtype == SVL_BF16, adjacent, form, (hipStream_t)stream));
    return SVL_OK;
}

svl_status svl_attention_plan_create(svl_ctx *ctx, const svl_attention_shape *shape,
                                     const int64_t *q_offsets, const int64_t *kv_offsets,
                                     const int64_t *prefix, int32_t documents,
                                     svl_attention_plan **out) {
    std::vector<AttnWork> work;
    std::vector<AttnJoin> join;
    std::vector<AttnTiles> tiles;
    auto build = [&](svl_attention_plan &plan) {
        if (!shape || !q_offsets) return fail(SVL_USAGE, "shape or offsets are null");
        if (documents < 0) return fail(SVL_USAGE, "document count is negative");
        if (shape->dtype != SVL_F32 && shape->dtype != SVL_BF16)
            return fail(SVL_UNSUPPORTED, "attention of type %d: F32 and BF16 are supported",
                        shape->dtype);
        if (shape->num_heads <= 0 || shape->num_kv_heads <= 0 ||
            shape->num_heads % shape->num_kv_heads)
            return fail(SVL_USAGE, "%lld heads are not a multiple of %lld key/value heads",
                        (long long)shape->num_heads, (long long)shape->num_kv_heads);
        if (shape->num_heads > 65536) return fail(SVL_LIMIT, "more than 65536 heads");
        if (shape->head_dim < 1 || shape->head_dim > 1024)
            return fail(SVL_UNSUPPORTED, "head dim %lld is outside 1..=1024",
                        (long long)shape->head_dim);
        const int64_t *ko = kv_offsets ? kv_offsets : q_offsets;
        ST_TRY(check_offsets(q_offsets, documents, "query"));
        ST_TRY(check_offsets(ko, documents, "key"));
        const int64_t G = shape->num_heads / shape->num_kv_heads;
        for (int32_t d = 0; d < documents; ++d) {
            if (prefix && prefix[d] < 0) return fail(SVL_USAGE, "prefix %d is negative", d);
            if ((q_offsets[d + 1] - q_offsets[d]) * G > INT32_MAX - 1024)
                return fail(SVL_LIMIT, "document %d: more than 2^31 query rows of heads", d);
        }
        plan.shape = *shape;
        plan.shape.window = shape->window < 0 ? -1 : std::min<int64_t>(shape->window, INT32_MAX);
        return fill_attention(plan, q_offsets, ko, prefix, documents, work, join, tiles);
    };
    return make_plan(ctx, out, build, [&](svl_attention_plan &plan) {
        ST_TRY(upload(work, &plan.work));
        ST_TRY(upload(join, &plan.join));
        return upload(tiles, &plan.key_tiles);
    });
}

svl_status svl_attention_plan_destroy(svl_attention_plan *plan) {
    if (!plan) return SVL_OK;
    OnDevice on(plan->device);
    delete plan;
    return SVL_OK;
}

int64_t svl_attention_plan_workspace(const svl_attention_plan *plan) {
    return plan ? plan->workspace : 0;
}

svl_status svl_masked_attention(const svl_attention_plan *plan, const svl_attention_args *args,
                                void *workspace, size_t workspace_bytes, void *stream) {
    if (!plan || !args) return fail(SVL_USAGE, "plan or arguments are null");
    const svl_attention_args &x = *args;
    const svl_attention_shape &sh = plan->shape;
    if (!std::isfinite(x.scale)) return fail(SVL_USAGE, "attention scale must be finite");
    if (!std::isfinite(x.soft_cap) || x.soft_cap < 0)
        return fail(SVL_USAGE, "score cap must be finite and not negative");
    if (plan->n_work == 0) return SVL_OK;
    if (!x.q || !x.out || (plan->kv_rows > 0 && (!x.k || !x.v)))
        return fail(SVL_USAGE, "rows are null");
    ST_TRY(check_strides(x.q_token_stride, x.q_head_stride));
    ST_TRY(check_strides(x.k_token_stride, x.k_head_stride));
    ST_TRY(check_strides(x.v_token_stride, x.v_head_stride));
    ST_TRY(check_strides(x.out_token_stride, x.out_head_stride));
    if (!rows_apart(plan->q_rows, sh.num_heads, x.out_token_stride, x.out_head_stride, sh.head_dim))
        return fail(SVL_USAGE, "output rows overlap");
    const int64_t size = sh.dtype == SVL_BF16 ? 2 : 4;
    if (!aligned(x.q, size) || !aligned(x.k, size) || !aligned(x.v, size) ||
        !aligned(x.out, size) || !aligned(x.lse, 4) || !aligned(x.slopes, 4))
        return fail(SVL_USAGE, "rows are not aligned to their type");
    if (plan->workspace > 0) {
        if (!workspace || workspace_bytes < (size_t)plan->workspace)
            return fail(SVL_USAGE, "workspace of %zu bytes, %lld are needed", workspace_bytes,
                        (long long)plan->workspace);
        if (!aligned(workspace, 16)) return fail(SVL_USAGE, "workspace is not aligned to 16 bytes");
    }
    MaskedArgs a{};
    a.q = x.q;
    a.k = x.k;
    a.v = x.v;
    a.out = x.out;
    a.lse = x.lse;
    a.q_tok = x.q_token_stride;
    a.q_head = x.q_head_stride;
    a.k_tok = x.k_token_stride;
    a.k_head = x.k_head_stride;
    a.v_tok = x.v_token_stride;
    a.v_head = x.v_head_stride;
    a.o_tok = x.out_token_stride;
    a.o_head = x.out_head_stride;
    a.heads = (int32_t)sh.num_heads;
    a.kv_heads = (int32_t)sh.num_kv_heads;
    a.hd = (int32_t)sh.head_dim;
    a.causal = sh.causal != 0;
    a.window = (int32_t)sh.window;
    a.scale = x.scale;
    a.cap = x.soft_cap;
    a.slopes = x.slopes;
    a.work = plan->work;
    a.n_work = plan->n_work;
    a.join = plan->join;
    a.n_join = plan->n_join;
    a.join_vectors = plan->join_vectors;
    a.join_parts = plan->join_parts;
    a.partial = (float *)workspace;
    a.planes = (char *)workspace + plan->planes_at;
    a.tiles = plan->key_tiles;
    a.n_tiles = plan->n_tiles;
    OnDevice on(plan->device);
    HIP_TRY(on.err);
    HIP_TRY(launch_masked_attention(a, sh.dtype == SVL_BF16, plan->tiles, (hipStream_t)stream));
    return SVL_OK;
}

}  // extern "C"
