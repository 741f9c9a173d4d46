// Entry points of the attention over a cache in pages: what they check, which kernels they launch, and how large a workspace is.
#include <hip/hip_runtime.h>
#include <cmath>
#include "attention_paged_launch.hpp"
#include "cache.hpp"
#include "launch.hpp"

using namespace sddmm;

namespace {

// How a call's rows and keys are dealt out.
struct Deal {
    int64_t rows = 0;  // of all sequences
    bool token = true; // the kernel for few rows
    int tiles = 1;     // of 16 rows to a workgroup of it
    int tile = 128;    // rows of a workgroup of the kernel for many
    int64_t slots = 0, max_tiles = 0, grid = 0, splits = 1, chunk = 1;
    int64_t few_rows = 0, few_grid = 0, few_splits = 0;  // sequences of few rows beside others: rows at most, workgroups and pieces
    int64_t part_o = 0, part_ml = 0, few_o = 0, few_ml = 0, bytes = 0;  // where parts lie in the workspace, and those of sequences of few rows beside others
};

Deal deal(const sddmm_attention_desc &d)
{
    Deal r;
    const int64_t group = d.n_heads / d.n_kv_heads, packed = d.max_q * group;
    r.rows = rows_of(d);
    if (r.rows == 0) return r;
    // (us with the border at 32 / 64 / 128 rows, 8 key heads of 128: 16 users of up to 3000 keys, 36 and 64 rows over 8 bits 51 / 41 / 42 and 52 / 42 / 42, 96 and 128 rows 53 / 53 / 60 and
    // 56 / 56 / 77; over 16 bits 36 and 64 rows 44 / 46 / 46 and 44 / 47 / 47, 128 rows 49 / 49 / 88; one user of 8000 keys, 64 and 128 rows over 8 bits 22 / 22 / 22 and 28 / 28 / 25, over 16 bits
    // 20 / 22 / 22 and 25 / 25 / 25)
    r.token = packed <= 64;
    r.tiles = packed <= 16 ? 1 : 2;
    // Sequences of few rows among those of many, as far as numbers tell: packed ones whose longest is four times the mean (us in one launch and with tiles of rows for all, 32 heads over 8 of 128:
    // 32 sequences, up to 4000 keys, 2000 rows, the longest 8, 12 and 15 times the mean 218 and 231, 173 and 206, 141 and 158, 1000 rows, 31 times, 147 and 200; 8 sequences, up to 2000 keys, 1000
    // rows, 3 times 68 and 57, 5 to 8 times, where a few long tiles are most of the work, 82 to 84 and 67 to 74).
    const bool mixed = !r.token && d.type != SDDMM_TYPE_F32 && d.q_ptr && group <= 32 && (double)d.max_q * d.n_seq >= 4. * d.q_rows;
    // Many rows: 256 to a workgroup, which share the codes that it makes operands of, where there are 128 workgroups of them and long heads (us with 256 and 128: 2048 tokens behind
    // 14,336, 16 heads over 2 of 128, 8 bits 317 and 360; 1024 behind 7168, 32 over 8 167 and 177; a prompt of 4096, 32 over 8, 16 bits 147 and 164; 2048, 16 over 4 62 and 62; 128 behind
    // 8064 50 and 39; 16 of 300 tokens, heads of 64 54 and 43).
    if (!r.token && !mixed && d.type != SDDMM_TYPE_F32 && d.head_dim > 64 && (d.q_ptr ? r.rows * group / 256 + d.n_seq : div_up(packed, 256) * d.n_seq) * d.n_kv_heads >= 128) r.tile = 256;
    const int64_t few = r.token ? 16 * r.tiles : r.tile;
    r.max_tiles = div_up(packed, few);
    r.slots = r.max_tiles == 1 && r.token ? d.n_seq : d.q_ptr ? r.rows * group / few + d.n_seq : r.max_tiles * d.n_seq;
    const int64_t workgroups = r.slots * d.n_kv_heads;
    // keys that a tile's rows can see, in tiles of 32
    const int64_t span = d.window_left >= 0 && d.window_right >= 0 && !d.prefix ? (int64_t)d.window_left + d.window_right + std::min<int64_t>(d.max_q, few) : d.max_k;
    const int64_t key_tiles = std::max<int64_t>(1, std::min<int64_t>(div_up(d.max_k, 32), span / 32 + 2));
    if (r.token) {
        // Pieces, so that there are 512 workgroups, two to a compute unit; where there are as many without pieces, eight times as many, which evens out the lengths of caches (us with
        // 512 / 1024 / 4096: 64 users of up to 8192 keys, 8 key heads of 128 126 / 145 / 120; 512 / 1024: 4 of up to 32,768, 2 key heads 16.8 / 18.5; 16 of a window of 2048, 4 of 64
        // 16.5 / 20.5; 8 of 6000, 8 tokens of 4 heads for each of 4 22 / 33).  Of 256 keys and more, or of 128 while these are so few that the join is short (of 128 and of 256 keys: one
        // user, 1501 keys, 10.2 / 10.4; 16,384 keys, 8 heads over 2 11.5 / 12.1; 2 users, 4 tokens, 8192 keys 11.9 / 12.6; 32,768 keys 14.8 / 13.1; 16 tokens, 16 heads, 8192 keys 18.6 / 15.9).
        if (workgroups >= 512) {
            r.splits = std::min(div_up(4096, workgroups), div_up(key_tiles, 32));
        } else {
            const int64_t fine = std::min(div_up(key_tiles, 4), std::min<int64_t>(128, 8192 / (r.rows * d.n_heads)));
            r.splits = std::min(std::min(div_up(512, workgroups), std::max(fine, div_up(key_tiles, 8))), (int64_t)256);
        }
        r.chunk = div_up(key_tiles, r.splits);
        r.splits = div_up(key_tiles, r.chunk);
    } else {
        // As many pieces as fill the card (rows of packed sequences counted without the slots that few of them leave empty where most sequences have few rows: three pieces of prompts beside
        // 29 tokens, 1053 rows of 32 heads over 8, up to 4096 keys, in whole and in 2, 3 and 4 pieces 153, 111, 126 and 132 us).
        const int64_t filled = mixed ? std::max<int64_t>(1, r.rows * group / r.tile) * d.n_kv_heads : workgroups;
        r.splits = std::max<int64_t>(1, std::min(std::min(div_up(r.tile == 256 ? 256 : 512, filled), div_up(key_tiles, 8)), (int64_t)256));
    }
    r.grid = workgroups * r.splits;
    if (mixed) {
        r.few_rows = group <= 16 ? 16 : 32;
        const int64_t caches = (int64_t)d.n_seq * d.n_kv_heads;
        // (beside the others: a workgroup for each compute unit, pieces of up to 4096 keys; 512 and 1024 workgroups 113 and 120 us where 256 take 111)
        // No more than 4096 workgroups, where there are several to a cache: their parts (68 MB for heads of 128) would grow with the longest length that a caller allows for.
        r.few_splits = std::max<int64_t>(1, std::min(std::min(std::max(div_up(256, caches), std::min(div_up(key_tiles, 128), 4096 / caches)), div_up(key_tiles, 4)), (int64_t)256));
        r.chunk = div_up(key_tiles, r.few_splits);
        r.few_splits = div_up(key_tiles, r.chunk);
        r.few_grid = caches * r.few_splits;
    }
    auto place = [&](int64_t parts, int64_t rows, int64_t &o, int64_t &ml) {
        o = r.bytes, ml = o + padded(parts * rows * d.head_dim * (int64_t)sizeof(float));
        r.bytes = ml + padded(parts * rows * (int64_t)sizeof(float2));
    };
    if (r.splits > 1) place(r.splits, r.rows * d.n_heads, r.part_o, r.part_ml);
    if (r.few_splits > 1) place(r.few_splits, d.n_seq * r.few_rows * d.n_kv_heads, r.few_o, r.few_ml);
    return r;
}

int check(const char *who, const sddmm_attention_desc *desc, const sddmm_cache_desc *cache)
{
    if (!desc) return fail(SDDMM_ERR_ARG, "%s: NULL description", who);
    sddmm_attention_desc d = *desc;  // (keys are the cache's)
    d.k_seq = d.v_seq = d.k_head = d.v_head = d.k_rows = 0, d.k_row = d.v_row = 128;
    if (int rc = check_desc(who, &d)) return rc;
    return check_cache(who, d, cache);
}

}  // namespace

extern "C" {

int sddmm_attention_paged_workspace_bytes(const sddmm_attention_desc *desc, const sddmm_cache_desc *cache, int64_t *bytes)
{
    if (int rc = check("sddmm_attention_paged_workspace_bytes", desc, cache)) return rc;
    if (bytes) *bytes = deal(held(*desc)).bytes;
    return SDDMM_OK;
}

int sddmm_attention_paged(const sddmm_attention_desc *desc, const sddmm_cache_desc *cache, const void *d_q, void *d_out, float *d_lse,
                          void *d_workspace, int64_t workspace_bytes, void *stream)
{
    const char *who = "sddmm_attention_paged";
    if (int rc = check(who, desc, cache)) return rc;
    const sddmm_attention_desc d = sddmm::held(*desc);
    const Deal r = deal(d);
    if (r.rows == 0) return SDDMM_OK;
    if (!d_q || !d_out) return fail(SDDMM_ERR_ARG, "%s: NULL device pointer", who);
    if (!apart(d, d.o_seq, d.o_row, d.o_head, d.q_ptr ? 1 : d.n_seq, d.q_ptr ? d.q_rows : d.max_q, d.n_heads)) return fail(SDDMM_ERR_ARG, "%s: rows of the result overlap", who);
    if ((uintptr_t)d_lse & 3u) return fail(SDDMM_ERR_ARG, "%s: lse must be aligned to its elements", who);
    if (!aligned({d_q, d_out})) return fail(SDDMM_ERR_ARG, "%s: pointers must be 16-byte aligned", who);
    if (r.bytes > 0 && (!d_workspace || workspace_bytes < r.bytes || ((uintptr_t)d_workspace & 255u)))
        return fail(SDDMM_ERR_ARG, "%s: a workspace of %lld bytes, 256-byte aligned, is needed (got %lld)", who, (long long)r.bytes, (long long)workspace_bytes);
    const int64_t join = (r.splits > 1 ? attention_paged_join_grid(r.rows * d.n_heads, (int)r.splits, d.head_dim) : 0) +
                         (r.few_splits > 1 ? attention_paged_join_grid(d.n_seq * r.few_rows * d.n_kv_heads, (int)r.few_splits, d.head_dim) : 0);
    if (!launchable(r.grid + r.few_grid, 512) || !launchable(join, 512))
        return fail(SDDMM_ERR_RANGE, "%s: too many rows and heads for one launch", who);
    if (in_place_of({d_out, d_lse}, {d_q, cache->k, cache->v, cache->k_scale, cache->v_scale}) || (const void *)d_lse == d_out)
        return fail(SDDMM_ERR_ARG, "%s: a result is in an operand's or the other result's place", who);

    AttnArgs a = arguments(d);
    a.q = d_q, a.out = d_out, a.lse = d_lse;
    char *const ws = (char *)d_workspace;
    a.part_o = (float *)(ws + r.part_o), a.part_ml = (float2 *)(ws + r.part_ml);
    a.n_slots = (int)r.slots, a.max_tiles = (int)r.max_tiles, a.n_split = a.n_part = (int)r.splits, a.chunk = (int)r.chunk;
    a.few_rows = (int)r.few_rows;
    const CacheArgs c = cache_arguments(d, *cache);
    const hipStream_t st = (hipStream_t)stream;
    const int held = held_as(d, *cache);
    hipError_t e;
    AttnArgs few = a;
    if (r.few_grid > 0) {
        few.n_slots = d.n_seq, few.max_tiles = 1, few.n_split = few.n_part = (int)r.few_splits;
        few.part_o = (float *)(ws + r.few_o), few.part_ml = (float2 *)(ws + r.few_ml), few.not_ml = r.splits > 1 ? a.part_ml : nullptr;
        e = launch_attention_paged_mixed(a, few, c, d.type, held, (unsigned)r.grid, (unsigned)r.few_grid, st);
    } else {
        e = r.token ? launch_attention_paged_token(a, c, d.type, held, r.tiles, (unsigned)r.grid, st) : launch_attention_paged_forward(a, c, d.type, held, r.tile, (unsigned)r.grid, st);
    }
    if (e == hipSuccess && join > 0) e = launch_attention_paged_join(a, r.few_splits > 1 ? &few : nullptr, d.type, st);
    if (e != hipSuccess) return fail(SDDMM_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
    return SDDMM_OK;
}

}  // extern "C"
