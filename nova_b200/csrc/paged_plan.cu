// Host side of the paged calls: the plan of one step of a batch of requests
// (lengths, pages, work lists), built without a GPU into one int32 array that
// the caller copies to the device once per step and every layer reads.  About
// 40 us for 2048 new tokens over 30011 or 64 requests of one token.
#include <new>
#include <vector>

#include "paged.cuh"

namespace {

using nova::fail;
using namespace nova::paged;

struct Builder {
    const nova_paged_plan_args& a;
    std::vector<int32_t> v;
    int64_t at() {                       // sections start on 16 bytes
        while (v.size() % 4) v.push_back(0);
        return int64_t(v.size());
    }
    template <typename T>
    void put(const T& rec) {
        const int32_t* p = reinterpret_cast<const int32_t*>(&rec);
        v.insert(v.end(), p, p + sizeof(T) / 4);
    }
};

// Lengths, page numbers and tail buffers of the step.
int check_requests(const nova_paged_plan_args& a) {
    if (a.seqs < 1 || a.seqs > (1 << 20)) return fail(NOVA_ERR_INVALID, "plan: seqs=%lld", (long long)a.seqs);
    if (a.kv_heads < 1 || a.q_heads < 1 || a.q_heads % a.kv_heads)
        return fail(NOVA_ERR_INVALID, "plan: q_heads %lld is not a multiple of kv_heads %lld", (long long)a.q_heads,
                    (long long)a.kv_heads);
    if (a.kv_heads > 1024 || a.q_heads > 16384 || a.sms < 1)
        return fail(NOVA_ERR_INVALID, "plan: kv_heads, q_heads or sms out of range");
    if (a.n_windows < 0 || a.n_windows > NOVA_PAGED_MAX_WINDOWS)
        return fail(NOVA_ERR_INVALID, "plan: at most %d windows, got %lld", NOVA_PAGED_MAX_WINDOWS,
                    (long long)a.n_windows);
    for (int64_t w = 0; w < a.n_windows; ++w)
        if (a.windows[w] < 0 || a.windows[w] > (1ll << 30)) return fail(NOVA_ERR_INVALID, "plan: window out of range");
    const int64_t lim = (1ll << 31) - 4096;
    int64_t tokens = 0, rows = 0;
    std::vector<std::pair<int64_t, int64_t>> bufs, written;
    for (int64_t i = 0; i < a.seqs; ++i) {
        const int64_t q = a.q_lens[i], kv = a.kv_lens[i], start = kv - q, np = a.page_off[i + 1] - a.page_off[i];
        if (q < 0 || kv < q || kv >= lim)
            return fail(NOVA_ERR_INVALID, "plan: request %lld has %lld new tokens and length %lld", (long long)i,
                        (long long)q, (long long)kv);
        if (a.page_off[i] < 0 || np < kv / PT)
            return fail(NOVA_ERR_INVALID, "plan: request %lld of length %lld has %lld pages, %lld are needed",
                        (long long)i, (long long)kv, (long long)np, (long long)(kv / PT));
        if (a.page_off[i + 1] >= lim) return fail(NOVA_ERR_INVALID, "plan: too many pages");
        for (int64_t j = 0; j < np; ++j) {
            const int64_t p = a.pages[a.page_off[i] + j];
            if (p < 0 || p >= lim) return fail(NOVA_ERR_INVALID, "plan: request %lld has page %lld", (long long)i, (long long)p);
            if (j >= start / PT && j < kv / PT) written.push_back({p, i});
        }
        const bool takes = start % PT != 0, leaves = kv % PT != 0, same = start / PT == kv / PT;
        if ((takes && (a.tail_in[i] < 0 || a.tail_in[i] >= lim)) || (leaves && (a.tail_out[i] < 0 || a.tail_out[i] >= lim)))
            return fail(NOVA_ERR_INVALID, "plan: request %lld needs a tail buffer", (long long)i);
        if (takes && leaves && same && a.tail_in[i] != a.tail_out[i])
            return fail(NOVA_ERR_INVALID, "plan: the open page of request %lld stays open: tail_out must be tail_in", (long long)i);
        if (takes && leaves && !same && a.tail_in[i] == a.tail_out[i])
            return fail(NOVA_ERR_INVALID, "plan: request %lld opens another page: tail_out must differ from tail_in", (long long)i);
        if (takes) bufs.push_back({a.tail_in[i], i});
        if (leaves) bufs.push_back({a.tail_out[i], i});
        if (a.read_from && (a.read_from[i] < 0 || a.read_from[i] > kv))
            return fail(NOVA_ERR_INVALID, "plan: read_from %lld of request %lld outside [0, %lld]",
                        (long long)a.read_from[i], (long long)i, (long long)kv);
        tokens += q;
        rows += kv - (a.read_from ? a.read_from[i] : start / PT * PT);
        if (tokens >= lim || rows >= lim || tokens * (a.q_heads + 2 * a.kv_heads + 12) >= lim)
            return fail(NOVA_ERR_UNSUPPORTED, "plan: too many tokens in one step");
    }
    std::sort(bufs.begin(), bufs.end());
    for (size_t i = 1; i < bufs.size(); ++i)
        if (bufs[i].first == bufs[i - 1].first && bufs[i].second != bufs[i - 1].second)
            return fail(NOVA_ERR_INVALID, "plan: two requests share tail buffer %lld", (long long)bufs[i].first);
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
        if (written[i].first == written[i - 1].first)
            return fail(NOVA_ERR_INVALID, "plan: page %lld would be written twice", (long long)written[i].first);
    return NOVA_OK;
}

// Blocks that the query rows [row0, row0 + nrows) of request i can see.
void seen_blocks(const nova_paged_plan_args& a, int64_t i, int64_t row0, int64_t nrows, int64_t window, int64_t* b0,
                 int64_t* b1) {
    const int64_t gq = a.q_heads / a.kv_heads, start = a.kv_lens[i] - a.q_lens[i];
    const int64_t first = start + row0 / gq, last = start + (row0 + nrows - 1) / gq;
    *b0 = window > 0 ? std::max<int64_t>(0, first - window + 1) / PT : 0;
    *b1 = last / PT + 1;
}

// Which kernel takes request i.  A tile of the few-rows kernel holds 16 query
// rows of a KV head, the tensor-core kernel's 256; the first starts and joins
// faster, the second reads the cache once.  16 requests of up to 4000 tokens:
// up to 32 rows each 64 us there, 88 in the other (four of 1000: 25 and 44); one of
// 8192 tokens, 64 rows: 47 and 29.
constexpr int64_t FEW_ROWS = 2 * ROWS_MAX;
bool few_rows(const nova_paged_plan_args& a, int64_t i) { return a.q_lens[i] * (a.q_heads / a.kv_heads) <= FEW_ROWS; }

// Work lists of the few-rows kernel: requests of up to 4 rows, whose tiles keep
// the weights' low parts at no cost, and of more.  Every tile's blocks are cut
// into splits of at least one block per warp (4), at most 32 per tile so that
// joining them stays short.  A CTA costs a few blocks' time to start and to join, so where splits
// of up to 48 blocks let all CTAs be resident at once (3 per SM) the smallest
// such size is taken; 16 requests of 8191 tokens: 70 us, 76 in splits of 16.
// Beyond that about four times as many CTAs as are resident even out ragged
// lengths (32 requests of 8000 to 32768 tokens: 225 us, 260 in one wave).
void rows_schedule(Builder& b, const nova_paged_schedule& s, bool more, nova_paged_rows& list) {
    const nova_paged_plan_args& a = b.a;
    const int64_t gq = a.q_heads / a.kv_heads;
    auto mine = [&](int64_t i) { return few_rows(a, i) && (a.q_lens[i] * gq > 4) == more; };
    int64_t most = 0, total = 0;
    for (int64_t i = 0; i < a.seqs; ++i)
        if (mine(i)) most = std::max(most, a.q_lens[i] * gq);
    list.rows_per_tile = !more ? 4 : most <= 8 ? 8 : ROWS_MAX;
    std::vector<int64_t> tiles;                // blocks of each tile
    for (int64_t i = 0; i < a.seqs; ++i)
        for (int64_t r = 0; mine(i) && r < a.q_lens[i] * gq; r += list.rows_per_tile) {
            int64_t b0, b1;
            seen_blocks(a, i, r, std::min(list.rows_per_tile, a.q_lens[i] * gq - r), s.window, &b0, &b1);
            tiles.push_back(b1 - b0);
            total += b1 - b0;
        }
    const int64_t resident = a.sms * 3;
    int64_t chunk = 4;
    for (; chunk <= 48; chunk += 4) {
        int64_t ctas = 0;
        for (int64_t n : tiles) ctas += (n + chunk - 1) / chunk * a.kv_heads;
        if (ctas <= resident) break;
    }
    if (chunk > 48) chunk = std::max<int64_t>(16, total * a.kv_heads / (resident * 4) / 4 * 4);
    list.off = b.at();
    int64_t q_start = 0;
    for (int64_t i = 0; i < a.seqs; q_start += a.q_lens[i++])
        for (int64_t r = 0; mine(i) && r < a.q_lens[i] * gq; r += list.rows_per_tile) {
            const int64_t n = std::min(list.rows_per_tile, a.q_lens[i] * gq - r);
            int64_t b0, b1;
            seen_blocks(a, i, r, n, s.window, &b0, &b1);
            const int64_t c = std::max(chunk, ((b1 - b0 + 31) / 32 + 3) / 4 * 4);
            const int64_t splits = (b1 - b0 + c - 1) / c;
            for (int64_t k = 0; k < splits; ++k) {
                RowsItem it{int(r), int(n), int(b0 + k * c), int(std::min(b1, b0 + (k + 1) * c)),
                            splits > 1 ? int(list.n_parts) : -1, int(k), int(splits), int(q_start),
                            int(a.kv_lens[i] - a.q_lens[i]), int(a.kv_lens[i]), int(a.page_off[i]),
                            a.kv_lens[i] % PT ? int(a.tail_out[i]) : 0, {-1, -1, -1, -1}};
                for (int w = 0; w < 4; ++w)
                    if (it.blk0 + w < std::min<int64_t>(it.blk1, a.kv_lens[i] / PT))
                        it.page[w] = int(a.pages[a.page_off[i] + it.blk0 + w]);
                b.put(it);
                ++list.n;
            }
            if (splits > 1) list.n_parts += splits;
        }
}

// Segments of the tensor-core kernel: the steps (128 keys) of all 256-row tiles
// in a row, request by request and head by head so that neighbouring CTAs read
// the same cache, cut so that no CTA takes more than a share; the smallest share
// that the SMs can hold is searched.  A segment costs about SEG_COST steps
// besides its own (its result, the pipeline's fill; taken as 2, 3 or 4 it gave times
// within 5 % of one another), and a tile is not cut into pieces below MIN_STEPS
// (64 tokens over 500 cached: 25.6 us with 1, 28.7 with 3; longer caches alike).
constexpr int64_t SEG_COST = 4, MIN_STEPS = 1;

struct Tile {
    int64_t seq, head, row0, nrows, b0, b1, q_start;
};

// Deals the tiles' steps out to CTAs of `share` each -> how many it takes.
// emit(tile, first block, end, new CTA).
template <typename Emit>
int64_t deal(const std::vector<Tile>& tiles, int64_t share, Emit&& emit) {
    int64_t ctas = 1, left = share;
    bool fresh = true;                         // nothing in this CTA yet
    for (const Tile& t : tiles)
        for (int64_t b0 = t.b0; b0 < t.b1;) {
            const int64_t steps = (t.b1 - b0 + 1) / 2, room = left - SEG_COST;
            int64_t take = std::min(steps, room);
            if (take < steps) take = std::min(take, steps - MIN_STEPS);
            if (take < std::min(steps, MIN_STEPS)) {
                if (!fresh) {
                    ++ctas;
                    left = share;
                    fresh = true;
                    continue;
                }
                take = steps;                  // a share too small for any cut: the whole tile
            }
            const int64_t end = std::min(t.b1, b0 + 2 * take);
            emit(t, b0, end, fresh);
            left -= take + SEG_COST;
            b0 = end;
            fresh = false;
        }
    return ctas - fresh;
}

void tile_schedule(Builder& b, nova_paged_schedule& s) {
    const nova_paged_plan_args& a = b.a;
    const int64_t gq = a.q_heads / a.kv_heads;
    std::vector<Tile> tiles;
    int64_t q_start = 0, total = 0;
    for (int64_t i = 0; i < a.seqs; q_start += a.q_lens[i++])
        for (int64_t h = 0; !few_rows(a, i) && h < a.kv_heads; ++h)
            for (int64_t r = 0; r < a.q_lens[i] * gq; r += 256) {
                Tile t{i, h, r, std::min<int64_t>(256, a.q_lens[i] * gq - r), 0, 0, q_start};
                seen_blocks(a, i, r, t.nrows, s.window, &t.b0, &t.b1);
                total += (t.b1 - t.b0 + 1) / 2 + SEG_COST;
                tiles.push_back(t);
            }
    if (tiles.empty()) return;
    auto none = [](const Tile&, int64_t, int64_t, bool) {};
    int64_t lo = std::max((total + a.sms - 1) / a.sms, MIN_STEPS + SEG_COST), hi = lo;
    while (deal(tiles, hi, none) > a.sms) hi *= 2;
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (deal(tiles, mid, none) <= a.sms) hi = mid;
        else lo = mid + 1;
    }
    std::vector<TileSeg> segs, first, more;    // segs in tile order; the CTAs' first ones go to the front
    std::vector<int64_t> opens;                // segs that open a CTA
    std::vector<TileJoin> joins;
    deal(tiles, hi, [&](const Tile& t, int64_t b0, int64_t end, bool fresh) {
        if (fresh) opens.push_back(int64_t(segs.size()));
        const bool cut = b0 != t.b0 || end != t.b1;
        if (cut && b0 == t.b0)
            joins.push_back(TileJoin{int(t.seq), int(t.head), int(t.row0), int(t.nrows), int(s.n_tile_parts), 0, 0, 0});
        if (cut) ++joins.back().n_parts;
        const int64_t kv = a.kv_lens[t.seq], off = a.page_off[t.seq];
        TileSeg g{int(t.head), int(t.row0), int(t.nrows), int(b0), int(end), cut ? int(s.n_tile_parts++) : -1, int(t.q_start),
                  int(kv - a.q_lens[t.seq]), int(kv), int(off), kv % PT ? int(a.tail_out[t.seq]) : 0, {-1, -1, -1, -1}, -1};
        for (int w = 0; w < 4; ++w)
            if (b0 + w < std::min(end, kv / PT)) g.page[w] = int(a.pages[off + b0 + w]);
        segs.push_back(g);
    });
    s.n_ctas = int64_t(opens.size());
    s.n_segs = int64_t(segs.size());
    opens.push_back(s.n_segs);
    for (int64_t c = 0; c < s.n_ctas; ++c)
        for (int64_t k = opens[c]; k < opens[c + 1]; ++k) {
            TileSeg& g = segs[k];
            if (k + 1 < opens[c + 1]) g.next = int(s.n_ctas + int64_t(more.size()) + (k > opens[c]));
            (k == opens[c] ? first : more).push_back(g);
        }
    s.segs_off = b.at();
    for (const TileSeg& g : first) b.put(g);
    for (const TileSeg& g : more) b.put(g);
    s.joins_off = b.at();
    s.n_joins = int64_t(joins.size());
    for (const TileJoin& j : joins) b.put(j);
}

// Where everything lies in the workspace of nova_paged_attention: the error
// word, the arrival counters (every launch leaves them at zero, so the schedules
// share them, with room for those of the largest), then the partials (dead after
// their launch, so the schedules share them too).  No schedule's partials may
// reach another's counters: launches of different schedules follow one another
// on one workspace, and only the plan's start zeroes it.
void place_workspace(nova_paged_plan_info& info) {
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    const int64_t heads = info.kv_heads;
    info.head_bytes = WS_HEAD;
    for (int64_t w = 0; w < info.n_windows; ++w) {
        int64_t at = WS_HEAD;
        for (nova_paged_rows& r : info.sched[w].rows) {
            r.counters_off = at;
            at += r.n_parts * heads * 4;
        }
        info.head_bytes = std::max(info.head_bytes, up(at));
    }
    info.workspace_bytes = info.head_bytes;
    for (int64_t w = 0; w < info.n_windows; ++w) {
        nova_paged_schedule& s = info.sched[w];
        int64_t at = info.head_bytes;
        for (nova_paged_rows& r : s.rows) {
            r.parts_off = at;
            at += up(r.n_parts * heads * r.rows_per_tile * PART * 4);
        }
        s.tile_parts_off = at;
        info.workspace_bytes = std::max(info.workspace_bytes, at + s.n_tile_parts * 256 * (D + 2) * 4);
    }
}

}  // namespace

extern "C" int nova_paged_plan(const nova_paged_plan_args* args, int32_t* out, int64_t capacity,
                               nova_paged_plan_info* info) {
    if (!args || !info) return fail(NOVA_ERR_INVALID, "plan: args and info must not be NULL");
    const nova_paged_plan_args& a = *args;
    if (!a.q_lens || !a.kv_lens || !a.page_off || !a.tail_in || !a.tail_out)
        return fail(NOVA_ERR_INVALID, "plan: NULL array");
    try {
        if (a.seqs > 0 && a.page_off[a.seqs] > 0 && !a.pages) return fail(NOVA_ERR_INVALID, "plan: NULL pages");
        if (int rc = check_requests(a)) return rc;
        *info = nova_paged_plan_info{};
        info->seqs = a.seqs;
        info->q_heads = a.q_heads;
        info->kv_heads = a.kv_heads;
        info->max_page = info->max_tail = info->max_pos = -1;
        Builder b{a, {}};
        info->seq_off = b.at();
        for (int64_t i = 0; i < a.seqs; ++i) {
            const int64_t kv = a.kv_lens[i], start = kv - a.q_lens[i];
            const bool takes = start % PT != 0, leaves = kv % PT != 0;
            Seq s{int(info->tokens), int(a.q_lens[i]), int(kv), int(a.page_off[i]), takes ? int(a.tail_in[i]) : 0,
                  leaves ? int(a.tail_out[i]) : 0, 0, 0};
            b.put(s);
            info->tokens += a.q_lens[i];
            if (a.q_lens[i]) info->max_pos = std::max(info->max_pos, kv - 1);
            if (takes) info->max_tail = std::max(info->max_tail, a.tail_in[i]);
            if (leaves) info->max_tail = std::max(info->max_tail, a.tail_out[i]);
        }
        info->page_off = b.at();
        for (int64_t j = 0; j < a.page_off[a.seqs]; ++j) {
            b.v.push_back(int32_t(a.pages[j]));
            info->max_page = std::max(info->max_page, a.pages[j]);
        }
        info->pos_off = b.at();
        for (int64_t i = 0; i < a.seqs; ++i)
            for (int64_t j = a.kv_lens[i] - a.q_lens[i]; j < a.kv_lens[i]; ++j) b.v.push_back(int32_t(j));
        info->open_off = b.at();
        int64_t first_row = 0;
        for (int64_t i = 0; i < a.seqs; first_row += a.q_lens[i++]) {
            const int64_t kv = a.kv_lens[i], start = kv - a.q_lens[i];
            for (int64_t j = std::max(start, kv / PT * PT); j < kv; ++j, ++info->n_open)
                b.put(OpenToken{int(first_row + j - start), int(j), int(a.tail_out[i]), 0});
        }
        info->write_off = b.at();
        int64_t row = 0;
        auto block = [&](int64_t i, int64_t g, int64_t first, int64_t out_row) {
            const int64_t kv = a.kv_lens[i], start = kv - a.q_lens[i];
            const bool full = (g + 1) * PT <= kv;
            return Block{int(g), int(first), int(kv), int(out_row), start % PT ? int(a.tail_in[i]) : 0,
                         kv % PT ? int(a.tail_out[i]) : 0, full ? int(a.pages[a.page_off[i] + g]) : -1, 0};
        };
        for (int64_t i = 0; i < a.seqs; row += a.q_lens[i++]) {
            const int64_t start = a.kv_lens[i] - a.q_lens[i];
            for (int64_t g = start / PT; a.q_lens[i] && (g + 1) * PT <= a.kv_lens[i]; ++g, ++info->n_write)
                b.put(block(i, g, start, row));
        }
        info->read_off = b.at();
        for (int64_t i = 0; i < a.seqs; ++i) {
            const int64_t kv = a.kv_lens[i], from = a.read_from ? a.read_from[i] : (kv - a.q_lens[i]) / PT * PT;
            for (int64_t g = from / PT; from < kv && g * PT < kv; ++g, ++info->n_read) b.put(block(i, g, from, info->read_rows));
            info->read_rows += kv - from;
        }
        info->n_windows = a.n_windows;
        for (int64_t w = 0; w < a.n_windows; ++w) {
            nova_paged_schedule& s = info->sched[w];
            s.window = a.windows[w];
            rows_schedule(b, s, false, s.rows[0]);
            rows_schedule(b, s, true, s.rows[1]);
            tile_schedule(b, s);
        }
        place_workspace(*info);
        info->ints = int64_t(b.v.size());
        if (out && capacity >= info->ints) memcpy(out, b.v.data(), b.v.size() * sizeof(int32_t));
        return NOVA_OK;
    } catch (const std::exception& e) {
        return fail(NOVA_ERR_INVALID, "plan: %s", e.what());
    }
}
