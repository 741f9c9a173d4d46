// Entry points of the dense attention: what they check, which kernels they launch, and how large a workspace is.
#include <hip/hip_runtime.h>
#include <cmath>
#include <cstring>
#include "internal.hpp"
#include "attention.hpp"
#include "attention_launch.hpp"
#include "launch.hpp"

using namespace sddmm;

namespace {

constexpr int64_t kMostRows = INT32_MAX;

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// head_dim as the kernels are made for (fp32, whose matrix instructions are a sixteenth as fast, by 32)
int64_t padded_dim(const sddmm_attention_desc &d) { return d.head_dim <= 32 && d.type == SDDMM_TYPE_F32 ? 32 : d.head_dim <= 64 ? 64 : 128; }

int element(int type) { return type == SDDMM_TYPE_F32 ? 4 : 2; }

bool strides_fit(const sddmm_attention_desc &d, int64_t seq, int64_t row, int64_t head, bool packed)
{
    const int64_t e = element(d.type), piece = 16 / e;
    return row >= d.head_dim && row < ((int64_t)1 << 23) / e && row % piece == 0 && head % piece == 0 && (packed || seq % piece == 0) &&
           head >= 0 && (packed || seq >= 0);
}

// Whether no two rows of an array that is written lie in each other's place (broadcast operands have strides of 0).
bool apart(const sddmm_attention_desc &d, int64_t seq, int64_t row, int64_t head, int64_t n_seq, int64_t n_rows, int64_t n_heads)
{
    std::pair<int64_t, int64_t> dims[3] = {{row, n_rows}, {head, n_heads}, {seq, n_seq}};
    if (n_seq == 0 || n_rows == 0) return true;
    std::sort(dims, dims + 3);
    int64_t extent = d.head_dim;
    for (const auto &[stride, n] : dims) {
        if (n <= 1) continue;
        if (stride < extent) return false;
        extent += (n - 1) * stride;
    }
    return true;
}

int check_desc(const char *who, const sddmm_attention_desc *p)
{
    if (!p) return fail(SDDMM_ERR_ARG, "%s: NULL description", who);
    const sddmm_attention_desc &d = *p;
    if (d.type != SDDMM_TYPE_F32 && d.type != SDDMM_TYPE_BF16 && d.type != SDDMM_TYPE_F16) return fail(SDDMM_ERR_ARG, "%s: unknown type %d", who, d.type);
    if (d.head_dim < 8 || d.head_dim > 128 || d.head_dim % 8)
        return fail(SDDMM_ERR_ARG, "%s: head_dim = %d is no multiple of 8 up to 128", who, d.head_dim);
    if (d.n_heads < 1 || d.n_kv_heads < 1 || d.n_heads % d.n_kv_heads || d.n_heads > 65536)
        return fail(SDDMM_ERR_ARG, "%s: %d query heads do not share %d key heads", who, d.n_heads, d.n_kv_heads);
    if (d.n_seq < 0 || d.max_q < 0 || d.max_k < 0 || d.shared_len < 0 || d.q_rows < 0 || d.k_rows < 0) return fail(SDDMM_ERR_ARG, "%s: negative size", who);
    if (d.window_left < -1 || d.window_right < -1) return fail(SDDMM_ERR_ARG, "%s: a window below -1", who);
    if (!std::isfinite(d.scale) || !(d.scale > 0.f)) return fail(SDDMM_ERR_ARG, "%s: scale must be finite and above 0", who);
    if (!std::isfinite(d.cap) || d.cap < 0.f) return fail(SDDMM_ERR_ARG, "%s: cap must be finite and not negative", who);
    if (d.cap > 0.f && !(d.scale / d.cap > 1e-15f && d.scale / d.cap < 1e15f && d.cap < 1e30f)) return fail(SDDMM_ERR_ARG, "%s: cap and scale are too far apart", who);
    if ((d.q_ptr && d.q_len) || (d.k_ptr && d.k_len)) return fail(SDDMM_ERR_ARG, "%s: lengths beside the pointers of packed sequences", who);
    if (!strides_fit(d, d.q_seq, d.q_row, d.q_head, d.q_ptr) || !strides_fit(d, d.k_seq, d.k_row, d.k_head, d.k_ptr) ||
        !strides_fit(d, d.v_seq, d.v_row, d.v_head, d.k_ptr) || !strides_fit(d, d.o_seq, d.o_row, d.o_head, d.q_ptr))
        return fail(SDDMM_ERR_ARG, "%s: strides must be multiples of 16 bytes, a row's from head_dim to 2^23 bytes", who);
    for (const void *p : {(const void *)d.q_ptr, (const void *)d.k_ptr, (const void *)d.q_len, (const void *)d.k_len, (const void *)d.prefix, (const void *)d.slopes})
        if ((uintptr_t)p & 3u) return fail(SDDMM_ERR_ARG, "%s: arrays of the description must be aligned to their elements", who);
    const int64_t rows = d.q_ptr ? d.q_rows : (int64_t)d.n_seq * d.max_q;
    if (rows > kMostRows || d.k_rows > kMostRows || (int64_t)d.shared_len + d.max_k > kMostRows / 2 || d.max_q > kMostRows / 2)
        return fail(SDDMM_ERR_RANGE, "%s: sizes beyond 32-bit positions", who);
    return SDDMM_OK;
}

// The description with the bounds that packed arrays give: no sequence has more rows or keys than all of them.  Tiles of a sequence then are at most those of the
// grid, and fit 32 bits as it does, whatever bound the caller names.
sddmm_attention_desc held(sddmm_attention_desc d)
{
    if (d.q_ptr) d.max_q = (int32_t)std::min<int64_t>(d.max_q, d.q_rows);
    if (d.k_ptr) d.max_k = (int32_t)std::min<int64_t>(d.max_k, d.k_rows);
    return d;
}

// Rows and keys of all sequences (0 where none can have any, whatever the arrays hold).
int64_t rows_of(const sddmm_attention_desc &d) { return d.n_seq == 0 || d.max_q == 0 ? 0 : d.q_ptr ? d.q_rows : (int64_t)d.n_seq * d.max_q; }
int64_t key_rows_of(const sddmm_attention_desc &d) { return d.n_seq == 0 || d.max_k == 0 ? 0 : d.k_ptr ? d.k_rows : (int64_t)d.n_seq * d.max_k; }

// How a call's rows are dealt out.
struct Deal {
    int64_t rows = 0;          // of all sequences
    bool token = false;        // the kernel for few rows
    int mapping = kRowsOfHead, tile = 128;
    int64_t slots = 0, max_tiles = 0, grid = 0, splits = 1;
    int64_t shared_slots = 0, shared_grid = 0, shared_splits = 0;
    int shared_tile = 128;
    int64_t parts = 1, part_bytes = 0, bytes = 0;
};

constexpr int64_t kFill = 512;  // workgroups that fill the card: 256 compute units, two each

// Pieces that the keys are cut into: so many that there are `fill` workgroups, each of `least` keys at least.
int64_t pieces(int64_t workgroups, int64_t keys, int64_t least, int64_t fill)
{
    return std::max<int64_t>(1, std::min(std::min(div_up(fill, std::max<int64_t>(workgroups, 1)), div_up(keys, least)), (int64_t)256));
}

Deal deal(const sddmm_attention_desc &d)
{
    Deal r;
    const int64_t group = d.n_heads / d.n_kv_heads, tile = 128, few = kTokenRows;
    r.rows = rows_of(d);
    // keys that a tile's rows can see
    const int64_t span = d.window_left >= 0 && d.window_right >= 0 && !d.prefix ? (int64_t)d.window_left + d.window_right + std::min<int64_t>(d.max_q, tile) : d.max_k;
    const int64_t keys = std::min<int64_t>(d.max_k, span), seqs = d.q_ptr ? 1 : d.n_seq, packed = d.max_q * group;
    // Tiles of 128 rows where that makes 1024 workgroups, else of 64 (us of the forward pass, causal, with 128, 64 and 32: 4096 tokens, 16 heads of 128,
    // bf16 111 / 102 / 123; 16 sequences of 512 40 / 51 / 88; 2048 tokens, 16 heads of 64 38 / 25 / 21, fp32 156 / 109 / 89; 2048, 4 of 128 42 / 29 / 23),
    // of one head or of pairs of few tokens and the heads that share a key head (not in packed sequences);
    for (int64_t tile : {128, 64}) {
        r.tile = (int)tile;
        r.mapping = group > 1 && d.max_q < tile && !d.q_ptr ? kRowsPacked : kRowsOfHead;
        r.max_tiles = div_up(r.mapping == kRowsPacked ? packed : d.max_q, tile);
        r.slots = d.q_ptr ? r.rows / tile + d.n_seq : r.max_tiles;
        r.grid = r.slots * seqs * d.n_kv_heads * (r.mapping == kRowsPacked ? 1 : group);
        if (r.grid >= 2 * kFill) break;
    }
    // or tiles of 32 pairs, each wave on keys of its own, where pairs are few or there would be less than 768 of 64 rows
    r.token = d.shared_len > 0 || packed <= few || r.grid < kFill * 3 / 2;
    if (r.token) {
        r.max_tiles = div_up(packed, few);
        r.slots = r.max_tiles == 1 ? d.n_seq : d.q_ptr ? r.rows * group / few + d.n_seq : r.max_tiles * d.n_seq;
        r.grid = r.slots * d.n_kv_heads;
        // Few workgroups: pieces of 256 keys, two for each wave (one user, 1501 keys, 32 heads over 8: with 64 / 128 / 256 / 512 12.9 / 13.3 / 12.6 / 12.9 us, most of it two launches); up to
        // 768 keys a second launch costs more than it saves.
        // Where each workgroup has a cache of its own four times as many even out their lengths (64 users of 284 to 8192 keys: 512 / 1024 / 2048 / 4096
        // workgroups 232 / 218 / 207 / 214 us), which short ones do not pay for with a second launch.
        // fp32 products take 16 times as long: shorter pieces, as many as there are compute units (two workgroups' tiles of long heads do not fit one), where half of those
        // would have none (us with the rule for 16 bits and this: one token, 16 heads over 4 of 128, 700 keys 34 and 16; 6 sequences of 362, 6 over 3 of 96 20 and 15; a
        // prompt of 400, 4 of 128 25 and 18; where half of them have work: 38 tokens behind 3014, 32 over 4 of 96 84 and 116).  On either side of that border, one token of 32 heads
        // over 8: 120 workgroups, heads of 128, 700 keys 35 and 28, 1500 63 and 42, 4000 126 and 90, of 64 14 (400 keys) and 14, 19 and 24, 31 and 31; 136 workgroups, heads of 128 36 and
        // 36, 67 and 62, 142 and 152, of 64 14 and 18, 20 and 25, 34 and 33 (heads of 64 gain up to some 96: 64 workgroups 19 and 15, 96 19 and 20).
        const bool few_slow = d.type == SDDMM_TYPE_F32 && d.shared_len == 0 && r.grid < kFill / 4;
        if (r.max_tiles == 1 && r.grid >= kFill) r.splits = pieces(r.grid, keys, 1024, 4 * kFill);
        else if (few_slow) r.splits = keys <= 256 ? 1 : pieces(r.grid, keys, 128, d.head_dim > 64 ? kFill / 2 - r.grid + 1 : kFill);
        else r.splits = keys <= 768 ? 1 : pieces(r.grid, keys, 256, d.shared_len > 0 ? kFill / 2 : kFill);
        r.grid *= r.splits;
    }
    r.parts = r.splits;
    if (d.shared_len > 0) {
        // Tiles of 64 rows up to 256 rows of a key head, and one workgroup of them for each compute unit beside the others' (48 users behind 16,000 keys: 128, 256, 512
        // of them 49, 38 to 46 and 46 us).
        r.shared_tile = r.rows * group <= 256 ? 64 : 128;
        r.shared_slots = div_up(r.rows * group, r.shared_tile);
        // Pieces of 256 keys, fp32 of 64 (5 sequences of 4 tokens behind 294 keys, 32 over 8 heads of 96 25 and 16; 4 behind 1000, 16 over 4 of 64 19 and 12).
        r.shared_splits = pieces(r.shared_slots * d.n_kv_heads, d.shared_len, d.type == SDDMM_TYPE_F32 ? 64 : 256, kFill / 2);
        r.shared_grid = r.shared_slots * d.n_kv_heads * r.shared_splits;
        r.parts += r.shared_splits;
    }
    if (r.parts > 1) {
        r.part_bytes = padded(r.parts * r.rows * d.n_heads * d.head_dim * (int64_t)sizeof(float));
        r.bytes = r.part_bytes + padded(r.parts * r.rows * d.n_heads * (int64_t)sizeof(float2));
    }
    return r;
}

// The same for the backward pass.
struct DealBack {
    int64_t rows = 0, key_rows = 0, q_slots = 0, q_tiles = 0, kv_slots = 0, kv_tiles = 0, q_grid = 0, kv_grid = 0, splits = 1, chunk = 1, slope_parts = 0;
    int q_rows = 128, keys = 128;  // of a dq and a dk, dv workgroup
    int64_t lse_at = 0, delta_at = 0, parts_at = 0, slopes_at = 0, bytes = 0;  // places in the workspace
};

DealBack deal_back(const sddmm_attention_desc &d)
{
    DealBack r;
    const int64_t group = d.n_heads / d.n_kv_heads;
    r.rows = rows_of(d);
    r.key_rows = key_rows_of(d);
    if (r.rows > 0) {
        // (dq: us of the backward pass with 128, 64 and 32 rows: 4096 tokens, 16 heads of 128 351 / 341 / 402; 16 sequences of 512 123 / 142 / 228;
        // 2048 tokens, 4 heads 101 / 82 / 66)
        for (int64_t rows : {128, 64, 32}) {
            r.q_rows = (int)rows;
            r.q_tiles = div_up(d.max_q, rows);
            r.q_slots = d.q_ptr ? r.rows / rows + d.n_seq : r.q_tiles;
            r.slope_parts = r.q_slots * (d.q_ptr ? 1 : d.n_seq);
            r.q_grid = r.slope_parts * d.n_heads;
            if (r.q_grid >= (rows == 128 ? 2 * kFill : kFill)) break;
        }
    }
    if (r.key_rows > 0) {
        // Work: rows of all heads that see a tile of 128 keys, of all tiles, at most.  That of uneven sequences is not known here: between the mean and the
        // longest length.
        const bool window = d.window_left >= 0 && d.window_right >= 0 && !d.prefix;
        const double mean = d.k_ptr ? (double)r.key_rows / d.n_seq : d.max_k, uneven = std::min(1., std::sqrt(mean / std::max(d.max_k, 1))) * (d.window_right == 0 && !window ? 0.5 : 1.);
        auto rows_that_see = [&](int64_t keys) { return group * (window ? std::min<int64_t>(d.max_q, (int64_t)d.window_left + d.window_right + keys) : d.max_q); };
        double work = rows_that_see(128) * uneven * div_up(r.key_rows, 128) * d.n_kv_heads;
        // Tiles of 128 keys; of 64, the waves of which share the rows, where the work of 128 is little (heads up to 64, since two workgroups' tiles of longer
        // ones do not fit a compute unit); of 32 where it is so little that most waves would have none.  us of forward and backward, causal, bf16, heads of 64,
        // with 128, 64 and 32: 2 sequences of 512, 12 heads (work 24,000) 45 / 43 / 42; 2 of 1024, 8 heads (65,000) 53 / 51 / 43, 8 over 2 55 / 53 / 54, capped
        // 68 / 66 / 76; 4 of 1024, 12 heads (200,000) 83 / 69 / 84; 5999 tokens in 3, 12 heads (700,000) 218 / 209 / 226; 16,000 in 8 (1.7 million) 442 / 475 / 538.
        // Heads of 128, with 128 and 32: 148 tokens in 3, 16 over 2, fp32 112 and 62; 228, 8 over 2, fp16 46 and 48; 2898, 8 over 1, bf16 220 and 276.
        const double few = group == 1 ? 98304. : 32768.;
        r.keys = work < few ? 32 : work < 1048576. && d.head_dim <= 64 ? 64 : 128;
        r.kv_tiles = div_up(d.max_k, r.keys);
        r.kv_slots = d.k_ptr ? r.key_rows / r.keys + d.n_seq : r.kv_tiles;
        // (held to what no launch takes, so that nothing passes 64 bits)
        const int64_t workgroups = std::min(r.kv_slots * (d.k_ptr ? 1 : d.n_seq), (int64_t)1 << 40) * d.n_kv_heads, most = rows_that_see(r.keys);
        work = most * uneven * div_up(r.key_rows, r.keys) * d.n_kv_heads;
        // A tile of keys that most rows see is cut where it would take more than 2.5 equal shares of all work.  A piece costs the time of some 650 rows, written
        // and read, so pieces of c rows cost 650 work / c and save half of c at the end: c = sqrt(1300 share).  us of the backward pass, bf16, causal, with
        // this and whole tiles: 8192 tokens, 16 heads over 4 of 128 1130 and 1850; 4096, 16 over 2 390 and 1550; 2048, 16 over 4 of 64 80 and 186; forward and
        // backward of 13 documents of 22 to 2281 tokens in all 8192 345 and 574; where whole tiles stay: 8192, 16 over 16 1015, in pieces 1090.
        const int64_t places = r.keys == 32 || (d.type == SDDMM_TYPE_F32 && d.head_dim > 64) ? kFill / 2 : kFill;
        const double share = work / places;
        if (most > 2.5 * share) {
            const bool slow = d.type == SDDMM_TYPE_F32;  // (its rows take sixteen times as long, its parts no longer)
            // At least 256 rows, fp32 64; four times as many where four waves share the rows of 32 keys, fp32 down to half of that where there is room for more workgroups
            // (us: 253 tokens, 2 heads over 1 of 128 79 and 69; 245, 12 over 3 78 and 72; everywhere: 500, 8 over 8 98 and 107, 1013 in 2, 4 over 2 of 32 67 and 71).
            const int64_t least = r.keys != 32 ? (slow ? 64 : 256) : slow ? std::min<int64_t>(256, std::max<int64_t>(128, most * workgroups / places)) : 1024;
            r.chunk = std::max<int64_t>((int64_t)std::sqrt((slow ? 100. : 1300.) * share), least);
            r.splits = std::max<int64_t>(1, std::min<int64_t>(div_up(most, r.chunk), 32));
        }
        r.chunk = std::max(r.chunk, div_up(most, r.splits));
        r.kv_grid = workgroups * r.splits;
    }
    r.delta_at = padded(r.rows * d.n_heads * 4);
    r.parts_at = 2 * r.delta_at;
    r.slopes_at = r.parts_at + (r.splits > 1 ? r.kv_grid * r.keys * padded_dim(d) * 8 : 0);
    r.bytes = r.slopes_at + (d.slopes ? padded(r.slope_parts * d.n_heads * 8) : 0);
    return r;
}

AttnArgs arguments(const sddmm_attention_desc &d)
{
    AttnArgs a{};
    a.q_seq = d.q_seq, a.q_row = d.q_row, a.q_head = d.q_head, a.k_seq = d.k_seq, a.k_row = d.k_row, a.k_head = d.k_head;
    a.v_seq = d.v_seq, a.v_row = d.v_row, a.v_head = d.v_head, a.o_seq = d.o_seq, a.o_row = d.o_row, a.o_head = d.o_head;
    a.q_ptr = d.q_ptr, a.k_ptr = d.k_ptr, a.q_len = d.q_len, a.k_len = d.k_len, a.prefix = d.prefix, a.slopes = d.slopes;
    a.rows = rows_of(d), a.key_rows = key_rows_of(d);
    a.head_dim = d.head_dim, a.n_heads = d.n_heads, a.n_kv_heads = d.n_kv_heads, a.group = d.n_heads / d.n_kv_heads;
    a.n_seq = d.n_seq, a.max_q = d.max_q, a.max_k = d.max_k, a.left = std::min(d.window_left, 1 << 30), a.right = std::min(d.window_right, 1 << 30),  // (positions are below)
    a.shared_len = d.shared_len;
    a.scale = d.scale, a.cap = d.cap;
    return a;
}

bool aligned(std::initializer_list<const void *> pointers)
{
    for (const void *p : pointers)
        if ((uintptr_t)p & 15u) return false;
    return true;
}

// Whether a result begins where an operand does (workgroups that are still to come read operands).
bool in_place_of(std::initializer_list<const void *> results, std::initializer_list<const void *> operands)
{
    for (const void *r : results)
        for (const void *o : operands)
            if (r && r == o) return true;
    return false;
}

int run_forward(const char *who, const sddmm_attention_desc *desc, const void *d_q, const void *d_shared_k, const void *d_shared_v, const void *d_k,
                const void *d_v, void *d_out, float *d_lse, void *d_workspace, int64_t workspace_bytes, void *stream)
{
    const sddmm_attention_desc d = held(*desc);
    const Deal r = deal(d);
    if (r.rows == 0) return SDDMM_OK;
    const bool keys = key_rows_of(d) > 0;
    if (!d_q || !d_out || (keys && (!d_k || !d_v)) || (d.shared_len && (!d_shared_k || !d_shared_v))) return fail(SDDMM_ERR_ARG, "%s: NULL device pointer", who);
    if (!apart(d, d.o_seq, d.o_row, d.o_head, d.q_ptr ? 1 : d.n_seq, d.q_ptr ? d.q_rows : d.max_q, d.n_heads)) return fail(SDDMM_ERR_ARG, "%s: rows of the result overlap", who);
    if ((uintptr_t)d_lse & 3u) return fail(SDDMM_ERR_ARG, "%s: lse must be aligned to its elements", who);
    if (!aligned({d_q, d_k, d_v, d_out, d_shared_k, d_shared_v})) return fail(SDDMM_ERR_ARG, "%s: pointers must be 16-byte aligned", who);
    if (r.bytes > 0 && (!d_workspace || workspace_bytes < r.bytes || ((uintptr_t)d_workspace & 255u)))
        return fail(SDDMM_ERR_ARG, "%s: a workspace of %lld bytes, 256-byte aligned, is needed (got %lld)", who, (long long)r.bytes, (long long)workspace_bytes);
    if (!launchable(r.grid + r.shared_grid, kAttentionThreads) || (r.parts > 1 && !launchable(attention_join_grid(r.rows * d.n_heads, (int)r.parts, d.head_dim), kAttentionThreads)))
        return fail(SDDMM_ERR_RANGE, "%s: too many rows and heads for one launch", who);
    if (in_place_of({d_out}, {d_q, d_k, d_v, d_shared_k, d_shared_v})) return fail(SDDMM_ERR_ARG, "%s: the result is in an operand's place", who);

    AttnArgs a = arguments(d);
    a.q = d_q, a.k = d_k, a.v = d_v, a.out = d_out, a.lse = d_lse, a.shared_k = d_shared_k, a.shared_v = d_shared_v;
    a.part_o = (float *)d_workspace, a.part_ml = (float2 *)((char *)d_workspace + r.part_bytes);
    a.n_slots = (int)r.slots, a.max_tiles = (int)r.max_tiles, a.n_split = (int)r.splits, a.part0 = 0, a.n_part = (int)r.parts;
    const hipStream_t st = (hipStream_t)stream;
    hipError_t e = hipSuccess;
    if (d.shared_len > 0) {
        AttnArgs b = a;
        b.n_slots = (int)r.shared_slots, b.n_split = (int)r.shared_splits, b.part0 = (int)r.splits;
        e = launch_attention_shared(b, a, d.type, r.shared_tile, (unsigned)r.shared_grid, (unsigned)r.grid, st);
    } else {
        e = r.token ? launch_attention_token(a, d.type, (unsigned)r.grid, st) : launch_attention_forward(a, d.type, r.mapping, r.tile, (unsigned)r.grid, st);
    }
    if (e == hipSuccess && r.parts > 1) e = launch_attention_join(a, d.type, st);
    if (e != hipSuccess) return fail(SDDMM_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
    return SDDMM_OK;
}

}  // namespace

extern "C" {

void sddmm_attention_desc_init(sddmm_attention_desc *desc)
{
    if (!desc) return;
    memset(desc, 0, sizeof *desc);
    desc->window_left = desc->window_right = -1;
}

int sddmm_attention_workspace_bytes(const sddmm_attention_desc *desc, int64_t *forward, int64_t *backward)
{
    if (int rc = check_desc("sddmm_attention_workspace_bytes", desc)) return rc;
    const sddmm_attention_desc d = held(*desc);
    if (forward) *forward = deal(d).bytes;
    if (backward) *backward = deal_back(d).bytes;
    return SDDMM_OK;
}

int sddmm_attention_forward(const sddmm_attention_desc *desc, const void *d_q, const void *d_k, const void *d_v, void *d_out, float *d_lse,
                            void *d_workspace, int64_t workspace_bytes, void *stream)
{
    const char *who = "sddmm_attention_forward";
    if (int rc = check_desc(who, desc)) return rc;
    if (desc->shared_len) return fail(SDDMM_ERR_ARG, "%s: shared_len is for sddmm_attention_shared", who);
    return run_forward(who, desc, d_q, nullptr, nullptr, d_k, d_v, d_out, d_lse, d_workspace, workspace_bytes, stream);
}

int sddmm_attention_shared(const sddmm_attention_desc *desc, const void *d_q, const void *d_shared_k, const void *d_shared_v, const void *d_k,
                           const void *d_v, void *d_out, float *d_lse, void *d_workspace, int64_t workspace_bytes, void *stream)
{
    const char *who = "sddmm_attention_shared";
    if (int rc = check_desc(who, desc)) return rc;
    if (desc->q_ptr) return fail(SDDMM_ERR_ARG, "%s: rows of packed sequences are not taken", who);
    if ((int64_t)desc->n_seq * desc->max_q * desc->n_heads > INT32_MAX) return fail(SDDMM_ERR_RANGE, "%s: too many rows", who);
    return run_forward(who, desc, d_q, d_shared_k, d_shared_v, d_k, d_v, d_out, d_lse, d_workspace, workspace_bytes, stream);
}

int sddmm_attention_backward(const sddmm_attention_desc *desc, const void *d_q, const void *d_k, const void *d_v, const void *d_out,
                             const float *d_lse, const void *d_dout, void *d_dq, void *d_dk, void *d_dv, float *d_dslopes, void *d_workspace,
                             int64_t workspace_bytes, void *stream)
{
    const char *who = "sddmm_attention_backward";
    if (int rc = check_desc(who, desc)) return rc;
    const sddmm_attention_desc d = held(*desc);
    if (d.shared_len) return fail(SDDMM_ERR_ARG, "%s: shared_len is for sddmm_attention_shared", who);
    if (d_dslopes && !d.slopes) return fail(SDDMM_ERR_ARG, "%s: gradients of slopes that are not there", who);
    const DealBack r = deal_back(d);
    if (r.rows == 0 && r.key_rows == 0 && !d_dslopes) return SDDMM_OK;
    if ((r.rows > 0 && (!d_q || !d_out || !d_lse || !d_dout || !d_dq)) || (r.key_rows > 0 && (!d_k || !d_v || !d_dk || !d_dv)))
        return fail(SDDMM_ERR_ARG, "%s: NULL device pointer", who);
    const int64_t q_seqs = d.q_ptr ? 1 : d.n_seq, k_seqs = d.k_ptr ? 1 : d.n_seq, q_rows = d.q_ptr ? d.q_rows : d.max_q, k_rows = d.k_ptr ? d.k_rows : d.max_k;
    if (!apart(d, d.q_seq, d.q_row, d.q_head, q_seqs, q_rows, d.n_heads) || !apart(d, d.k_seq, d.k_row, d.k_head, k_seqs, k_rows, d.n_kv_heads) ||
        !apart(d, d.v_seq, d.v_row, d.v_head, k_seqs, k_rows, d.n_kv_heads))
        return fail(SDDMM_ERR_ARG, "%s: rows of a gradient overlap", who);
    if (((uintptr_t)d_lse | (uintptr_t)d_dslopes) & 3u) return fail(SDDMM_ERR_ARG, "%s: lse and d_dslopes must be aligned to their elements", who);
    if (!aligned({d_q, d_k, d_v, d_out, d_dout, d_dq, d_dk, d_dv})) return fail(SDDMM_ERR_ARG, "%s: pointers must be 16-byte aligned", who);
    if (r.bytes > 0 && (!d_workspace || workspace_bytes < r.bytes || ((uintptr_t)d_workspace & 255u)))
        return fail(SDDMM_ERR_ARG, "%s: a workspace of %lld bytes, 256-byte aligned, is needed (got %lld)", who, (long long)r.bytes, (long long)workspace_bytes);
    if (!launchable(r.q_grid, kAttentionThreads) || !launchable(r.kv_grid, kAttentionThreads) ||
        !launchable(attention_sum_grid(r.kv_grid, (int)r.splits, r.keys, (int)padded_dim(d), d_dslopes ? d.n_heads : 0), kAttentionThreads))
        return fail(SDDMM_ERR_RANGE, "%s: too many rows and heads for one launch", who);
    if (in_place_of({d_dq, d_dk, d_dv}, {d_q, d_k, d_v, d_out, d_dout, d_lse}) || in_place_of({d_dq}, {d_dk, d_dv}) || in_place_of({d_dk}, {d_dv}))
        return fail(SDDMM_ERR_ARG, "%s: a gradient is in an operand's or another gradient's place", who);

    AttnArgs a = arguments(d);
    char *ws = (char *)d_workspace;
    a.q = d_q, a.k = d_k, a.v = d_v, a.out = (void *)d_out, a.lse = (float *)d_lse, a.dout = d_dout, a.dq = d_dq, a.dk = d_dk, a.dv = d_dv;
    a.stat_lse = (float *)(ws + r.lse_at), a.stat_delta = (float *)(ws + r.delta_at), a.part_o = (float *)(ws + r.parts_at);
    a.dslopes = d_dslopes, a.slope_part = d_dslopes ? (double *)(ws + r.slopes_at) : nullptr, a.slope_parts = (int)r.slope_parts;
    AttnArgs b = a;
    a.n_slots = (int)r.kv_slots, a.max_tiles = (int)r.kv_tiles, a.n_split = (int)r.splits, a.chunk = (int)std::min<int64_t>(r.chunk, INT32_MAX);
    b.n_slots = (int)r.q_slots, b.max_tiles = (int)r.q_tiles, b.n_split = 1;
    const hipError_t e = launch_attention_backward(a, b, d.type, (unsigned)r.kv_grid, r.keys, (unsigned)r.q_grid, r.q_rows, (hipStream_t)stream);
    if (e != hipSuccess) return fail(SDDMM_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
    return SDDMM_OK;
}

}  // extern "C"
