// C-ABI entry points for attention.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "host_common.hpp"
#include "../kernels/attention_args.hpp"

using namespace kmc_host;

namespace kmc_host {
#define KMC_DECLARE_ATTENTION(type)                                                                    \
    hipError_t launch_attention_forward_##type(const kmc::AttentionArgs &, int, bool, hipStream_t);     \
    hipError_t launch_attention_gradient_##type(const kmc::AttentionGradArgs &, int, bool, hipStream_t);
KMC_DECLARE_ATTENTION(0)
KMC_DECLARE_ATTENTION(1)
KMC_DECLARE_ATTENTION(2)
#undef KMC_DECLARE_ATTENTION
}  // namespace kmc_host

namespace {

constexpr int MAX_WIDTH = 256;
constexpr double MAX_SCALE = 2.0e38;  // times log2(e) still a number of fp32
constexpr int MAX_KEYS = 0x7fffffff - 1024;         // a tile behind the last key still has a number
int element_size(int type) { return type == KMC_FP32 ? 4 : 2; }

// Features that the kernels are compiled for.
int padded_width(int features) { return features <= 64 ? 64 : features <= 96 ? 96 : features <= 128 ? 128 : 256; }

// Whether rows can be read and written 16 bytes at a time: the address, and the stride of every dimension that is walked.  The tokens of a
// tile are read through one buffer descriptor, which wants rows that do not overlap and a tile that it can number in 31 bits.
struct Layout {
    int size;
    bool aligned = true;
    void operand(const void *p, int width)
    {
        if (p) aligned = aligned && aligned16(p) && width * size % 16 == 0;
    }
    void stride(int extent, int64_t stride)
    {
        if (extent > 1) aligned = aligned && stride * size % 16 == 0;
    }
    void tokens(int extent, int64_t stride, int width)
    {
        this->stride(extent, stride);
        if (extent > 1) aligned = aligned && stride >= width && stride < (1 << 24) / size;
    }
};

// The stride of tokens that a tile is read with.  That of a single token means nothing, and a small one would put the rows behind it on top of it.
int64_t token_stride(int extent, int64_t stride, int width) { return extent > 1 ? stride : width; }

int check_extents(int type, int l, int m, int n, int h, int g, int k, int o, float scale)
{
    if (type != KMC_FP32 && type != KMC_FP16 && type != KMC_BF16) return fail(KMC_ERR_INVALID_ARGUMENT, "element type %d is none of 0, 1, 2", type);
    if (l < 0 || m < 0 || n < 0 || h < 0 || g < 0) return fail(KMC_ERR_INVALID_ARGUMENT, "negative extent l=%d m=%d n=%d h=%d g=%d", l, m, n, h, g);
    if (n > MAX_KEYS) return fail(KMC_ERR_INVALID_ARGUMENT, "n=%d is beyond %d keys", n, MAX_KEYS);
    if (h > 0 && (g == 0 || h % g != 0)) return fail(KMC_ERR_INVALID_ARGUMENT, "h=%d is no multiple of g=%d", h, g);
    if (k < 1 || k > MAX_WIDTH || o < 1 || o > MAX_WIDTH)
        return fail(KMC_ERR_INVALID_ARGUMENT, "k=%d and o=%d must be in 1 .. %d", k, o, MAX_WIDTH);
    if (!(std::fabs(scale) <= MAX_SCALE)) return fail(KMC_ERR_INVALID_ARGUMENT, "scale must be finite and at most %g", MAX_SCALE);
    // rows of a head of keys over the batch, and rows times heads over the batch, are numbered in 31 bits
    if (static_cast<double>(l) * m * h > 2.0e9) return fail(KMC_ERR_INVALID_ARGUMENT, "l m h = %.0f is beyond 2e9 rows", static_cast<double>(l) * m * h);
    return KMC_OK;
}

// The scale to base 2 is kept positive, so that the largest score has the largest product; its sign moves into the queries.
void set_scale(float scale, float *scale_log2, float *query_factor)
{
    const float to_base_2 = std::fabs(scale) * 1.4426950408889634f;
    *scale_log2 = to_base_2 > 0.0f ? to_base_2 : 1.0f;
    *query_factor = to_base_2 > 0.0f ? (scale < 0.0f ? -1.0f : 1.0f) : 0.0f;
}

constexpr int ROWS_PER_WORKGROUP = 128;
constexpr int ROWS_OF_OWN_KEYS = 32;                // up to here every wave walks keys of its own

// How many parts the keys are cut into: the number with the smallest modelled time, in microseconds, fitted to sweeps of 1 .. 64 parts.
//   Tiles of rows (bound by the matrix cores): 128 rows meet 64 keys in 2.1 us per 128 features in 16 bits (fp32: 7 times as long) while two
//   workgroups share a CU, in 0.65 of that alone; a launch of more workgroups than fit waits for half of one at its end.
//   Beside another job (`beside_us` of its own) the two share the chip, and half of that job's time is in the way.  Rows of more than 256 bytes let one workgroup on a CU.
//   Single tokens (bound by memory): keys and values at 4.7 TB/s, but no workgroup faster than 4 us and 1.05 us per 128 keys of 128 features, and
//   3.5 us of its place for a workgroup; the launch waits for the last ones.
//   Joining the parts costs a launch, 5 us, and writing and reading a partial result per part.
// How many of the keys take part is not known here: it plans for all of them, whether there are lengths or not (an entry's own length is cut into the parts evenly).
// 1 token against 32000 keys of 8 heads: 257 us in 1 part, 34.8 in the 32 of this rule, 32.8 in the best number, 16; 4 x 200 queries against 3000 keys of 4 heads 47.3 in 4, the best;
// 256 x 1000 x 4 heads uncut 100, the best.  11 shapes with lengths of about 5, 25, 50, 75 and 100 % of the keys: above the best number of parts of each by 19, 5, 6, 6 and 5 %
// in the geometric mean (planned for three quarters of the keys where there are lengths: 32, 8, 7, 6 and 5 %).  8 shapes behind a prefix, with about 10, 50, 75 and 100 % of the own keys:
// 15, 7, 5 and 7 % above the best numbers of both (with all of the other job's time in the way and that plan 26, 14, 10 and 11 %).
double time_of_parts(int splits, int64_t base, int64_t rows_total, int64_t keys, bool own_keys, const kmc_attention_params *p, bool joined, double beside_us)
{
    const double size = element_size(p->type), width = padded_width(std::max(p->k, p->o));
    const int64_t workgroups = base * splits, least = own_keys ? 128 : 64;
    const double steps = static_cast<double>((keys + least * splits - 1) / (least * splits));
    const double join_us = (splits > 1 || joined ? rows_total * p->o * 8.0 / 4.0e6 * splits : 0.0) + (splits > 1 && !joined ? 5.0 : 0.0);
    if (own_keys) {
        const double one = 4.0 + steps * 1.05 * width / 128 * (p->type == KMC_FP32 ? 5.5 : 1.0);
        const double memory = keys * static_cast<double>(base) * (p->k + p->o) * size / 4.7e6;
        return join_us + std::max(memory, one) + workgroups * 3.5 / 512 + one * 0.3;
    }
    const double tile_us = 2.1 * width / 128 * (p->type == KMC_FP32 ? 7.0 : 1.0), one = steps * tile_us;
    if (beside_us > 0) return join_us + std::max(one, workgroups * one / 512 + 0.5 * beside_us);
    // rows of more than 256 bytes: one workgroup per CU, whole rounds of which the last one counts
    if (width * size > 256) return join_us + 0.55 * one * ((workgroups + 255) / 256);
    return join_us + (workgroups <= 256 ? 0.65 * one : workgroups <= 512 ? one : workgroups * one / 512 + 0.5 * one);
}

int choose_parts(int64_t base, int64_t rows_total, int64_t keys, bool own_keys, const kmc_attention_params *p, bool joined, double *us)
{
    static const int candidates[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 40, 48, 64};
    const double beside_us = *us;
    int best = 0;
    for (const int splits : candidates) {
        if (splits > 1 && (splits - 1) * (own_keys ? 128 : 64) >= keys) break;
        const double time = time_of_parts(splits, base, rows_total, keys, own_keys, p, joined, beside_us);
        if (best == 0 || time < *us) {
            *us = time;
            best = splits;
        }
    }
    return best;
}
static_assert(2 * 64 <= kmc::ATT_MAX_SLOTS, "the parts of two jobs");

// false: more workgroups than the kernels count (two jobs in 31 bits)
bool plan_job(kmc::AttentionJob *job, int first_segment, int last_segment, int64_t entries, int64_t rows, int keys, bool may_cut, bool joined,
              const kmc_attention_params *p, double *us)
{
    job->first_segment = first_segment;
    job->last_segment = last_segment;
    job->entries = static_cast<int>(entries);
    job->rows = static_cast<int>(rows);
    job->own_keys = rows <= ROWS_OF_OWN_KEYS;
    job->row_tiles = job->own_keys ? 1 : static_cast<int>((rows + ROWS_PER_WORKGROUP - 1) / ROWS_PER_WORKGROUP);
    const int64_t base = entries * p->g * job->row_tiles;
    job->splits = may_cut ? choose_parts(base, static_cast<int64_t>(p->l) * p->m * p->h, keys, job->own_keys, p, joined, us) : 1;
    const int64_t workgroups = base * job->splits;
    if (workgroups > 0x7fffff00ll / 2) return false;
    job->workgroups = static_cast<int>(workgroups);
    job->grid = static_cast<int>((workgroups + 7) / 8 * 8);
    job->slot = 0;
    job->partial = joined;
    return true;
}

struct Plan {
    kmc::AttentionArgs args;
    bool aligned, empty;
    int64_t bytes;              // of workspace
};

int64_t partial_bytes(const kmc::AttentionArgs &args) { return args.slots * args.rows_total * (4ll * args.partial_width + 8); }

int prepare(const kmc_attention_params *p, bool with_workspace, Plan *plan)
{
    if (!p) return fail(KMC_ERR_INVALID_ARGUMENT, "null parameter block");
    const int status = check_extents(p->type, p->l, p->m, p->n, p->h, p->g, p->k, p->o, p->scale);
    if (status != KMC_OK) return status;
    if (p->prefix_n < 0 || p->prefix_n > MAX_KEYS) return fail(KMC_ERR_INVALID_ARGUMENT, "prefix_n=%d is outside 0 .. %d", p->prefix_n, MAX_KEYS);
    const bool causal = p->causal != 0 || p->prefix_n > 0;              // own keys behind a prefix are met up to the query's own
    if (causal && p->key_mask) return fail(KMC_ERR_INVALID_ARGUMENT, "key_mask does not go with a prefix");
    const int64_t strides[] = {p->q_ls, p->q_ms, p->q_hs, p->key_ls, p->key_ns, p->key_gs, p->value_ls, p->value_ns, p->value_gs,
                               p->out_ls, p->out_ms, p->out_hs, p->key_mask_ls, p->key_mask_ns, p->prefix_key_ns, p->prefix_key_gs,
                               p->prefix_value_ns, p->prefix_value_gs};
    for (const int64_t stride : strides)
        if (stride < 0) return fail(KMC_ERR_INVALID_ARGUMENT, "negative stride");
    plan->bytes = 0;
    plan->empty = p->l == 0 || p->m == 0 || p->h == 0;
    if (plan->empty) return KMC_OK;
    if (causal && !p->key_lengths) return fail(KMC_ERR_INVALID_ARGUMENT, "a prefix, or causal, needs key_lengths");
    if (!p->q || !p->out) return fail(KMC_ERR_INVALID_ARGUMENT, "null q / out pointer");
    if (p->n > 0 && (!p->key || !p->value)) return fail(KMC_ERR_INVALID_ARGUMENT, "null key / value pointer");
    if (p->prefix_n > 0 && (!p->prefix_key || !p->prefix_value)) return fail(KMC_ERR_INVALID_ARGUMENT, "null prefix_key / prefix_value pointer");

    kmc::AttentionArgs &args = plan->args;
    args = kmc::AttentionArgs{};
    args.q = p->q; args.q_ls = p->q_ls; args.q_ms = p->q_ms; args.q_hs = p->q_hs;
    args.out = p->out; args.out_ls = p->out_ls; args.out_ms = p->out_ms; args.out_hs = p->out_hs;
    args.lse = p->lse;
    args.m = p->m; args.g = p->g; args.r = p->h / p->g; args.k = p->k; args.o = p->o;
    set_scale(p->scale, &args.scale_log2, &args.query_factor);
    args.rows_total = static_cast<int64_t>(p->l) * p->m * p->h;
    args.partial_width = (p->o + 3) / 4 * 4;

    const bool prefixed = p->prefix_n > 0;
    kmc::AttentionKeys &prefix = args.keys[0], &own = args.keys[prefixed ? 1 : 0];
    if (prefixed) {
        prefix.k = p->prefix_key; prefix.k_ns = token_stride(p->prefix_n, p->prefix_key_ns, p->k); prefix.k_gs = p->prefix_key_gs;
        prefix.v = p->prefix_value; prefix.v_ns = token_stride(p->prefix_n, p->prefix_value_ns, p->o); prefix.v_gs = p->prefix_value_gs;
        prefix.n = p->prefix_n;
    }
    own.k = p->key; own.k_ls = p->key_ls; own.k_ns = token_stride(p->n, p->key_ns, p->k); own.k_gs = p->key_gs;
    own.v = p->value; own.v_ls = p->value_ls; own.v_ns = token_stride(p->n, p->value_ns, p->o); own.v_gs = p->value_gs;
    own.lengths = p->key_lengths;
    own.mask = p->key_mask; own.mask_ls = p->key_mask_ls; own.mask_ns = p->key_mask_ns;
    own.n = p->n;
    own.causal = causal;

    Layout layout{element_size(p->type)};
    layout.operand(p->q, p->k);
    layout.operand(p->out, p->o);
    layout.stride(p->l, p->q_ls); layout.stride(p->m, p->q_ms); layout.stride(p->h, p->q_hs);
    layout.stride(p->l, p->out_ls); layout.stride(p->m, p->out_ms); layout.stride(p->h, p->out_hs);
    if (p->n > 0) {
        layout.operand(p->key, p->k);
        layout.operand(p->value, p->o);
        layout.stride(p->l, p->key_ls); layout.tokens(p->n, p->key_ns, p->k); layout.stride(p->g, p->key_gs);
        layout.stride(p->l, p->value_ls); layout.tokens(p->n, p->value_ns, p->o); layout.stride(p->g, p->value_gs);
    }
    if (prefixed) {
        layout.operand(p->prefix_key, p->k);
        layout.operand(p->prefix_value, p->o);
        layout.tokens(p->prefix_n, p->prefix_key_ns, p->k); layout.stride(p->g, p->prefix_key_gs);
        layout.tokens(p->prefix_n, p->prefix_value_ns, p->o); layout.stride(p->g, p->prefix_value_gs);
    }
    plan->aligned = layout.aligned && !(p->flags & KMC_FLAG_FORCE_SCALAR_ACCESS);

    const int64_t rows = static_cast<int64_t>(p->m) * args.r;
    bool fits = true;
    if (with_workspace && prefixed) {
        // the prefix as one problem of the rows of all entries, the entries' own keys as another
        double us = 0;
        fits = plan_job(&args.job[1], 1, 2, p->l, rows, p->n, true, true, p, &us);
        fits = fits && plan_job(&args.job[0], 0, 1, 1, p->l * rows, p->prefix_n, true, true, p, &us);
        args.job[1].slot = args.job[0].splits;
        args.slots = args.job[0].splits + args.job[1].splits;
    } else {
        double us = 0;
        fits = plan_job(&args.job[0], 0, prefixed ? 2 : 1, p->l, rows, p->n, with_workspace, false, p, &us);
        if (args.job[0].splits > 1) {
            args.job[0].partial = 1;
            args.slots = args.job[0].splits;
        }
    }
    if (!fits) return with_workspace ? prepare(p, false, plan) : fail(KMC_ERR_INVALID_ARGUMENT, "more workgroups than the kernels count");
    plan->bytes = partial_bytes(args);

    return KMC_OK;
}

constexpr int MAX_PARTS = 64;

// Parts that `base` workgroups of `steps` tiles each are cut into, by a model of the launch in microseconds: whole rounds of `slots` workgroups, each of
// which takes `step_us` per tile and 3 us around them, and the sum of the parts, which costs a launch and writing and reading `elements` per part.
int parts(int64_t base, int64_t slots, int64_t steps, double step_us, double elements)
{
    int best = 1;
    double best_us = 0;
    for (int splits = 1; splits <= MAX_PARTS && (splits == 1 || splits <= steps); ++splits) {
        const double rounds = static_cast<double>((base * splits + slots - 1) / slots);
        const double us = rounds * ((steps + splits - 1) / splits * step_us + 3.0) + (splits > 1 ? 5.0 + splits * elements * 8.0 / 4.0e6 : 0.0);
        if (splits == 1 || us < best_us) {
            best_us = us;
            best = splits;
        }
    }
    return best;
}

struct GradPlan {
    kmc::AttentionGradArgs args;
    bool aligned, empty;
    int64_t stats_bytes, shift_bytes, q_bytes, k_bytes, v_bytes;
    int64_t bytes() const { return stats_bytes + shift_bytes + q_bytes + k_bytes + v_bytes; }
};

int prepare(const kmc_attention_gradient_params *p, bool may_cut, GradPlan *plan)
{
    if (!p) return fail(KMC_ERR_INVALID_ARGUMENT, "null parameter block");
    const int status = check_extents(p->type, p->l, p->m, p->n, p->h, p->g, p->k, p->o, p->scale);
    if (status != KMC_OK) return status;
    if (p->key_entries != p->l && p->key_entries != 1) return fail(KMC_ERR_INVALID_ARGUMENT, "key_entries=%d is neither l=%d nor 1", p->key_entries, p->l);
    const int64_t strides[] = {p->q_ls, p->q_ms, p->q_hs, p->key_ls, p->key_ns, p->key_gs, p->value_ls, p->value_ns, p->value_gs, p->out_ls, p->out_ms,
                               p->out_hs, p->grad_out_ls, p->grad_out_ms, p->grad_out_hs, p->key_mask_ls, p->key_mask_ns};
    for (const int64_t stride : strides)
        if (stride < 0) return fail(KMC_ERR_INVALID_ARGUMENT, "negative stride");
    if (p->key_entries != p->l && (p->key_ls != 0 || p->value_ls != 0))
        return fail(KMC_ERR_INVALID_ARGUMENT, "one source for all entries has key_ls and value_ls 0");
    *plan = GradPlan{};
    plan->empty = p->l == 0 || p->m == 0 || p->h == 0;
    if (plan->empty) return KMC_OK;
    if (!p->q || !p->out || !p->grad_out || !p->lse || !p->grad_q) return fail(KMC_ERR_INVALID_ARGUMENT, "null q / out / grad_out / lse / grad_q pointer");
    if (p->n > 0 && (!p->key || !p->value || !p->grad_key || !p->grad_value))
        return fail(KMC_ERR_INVALID_ARGUMENT, "null key / value / grad_key / grad_value pointer");

    kmc::AttentionGradArgs &args = plan->args;
    args.q = p->q; args.q_ls = p->q_ls; args.q_ms = token_stride(p->m, p->q_ms, p->k); args.q_hs = p->q_hs;
    args.out = p->out; args.out_ls = p->out_ls; args.out_ms = p->out_ms; args.out_hs = p->out_hs;
    args.grad_out = p->grad_out; args.grad_out_ls = p->grad_out_ls; args.grad_out_ms = token_stride(p->m, p->grad_out_ms, p->o); args.grad_out_hs = p->grad_out_hs;
    args.lse = p->lse;
    kmc::AttentionKeys &keys = args.keys;
    keys.k = p->key; keys.k_ls = p->key_ls; keys.k_ns = token_stride(p->n, p->key_ns, p->k); keys.k_gs = p->key_gs;
    keys.v = p->value; keys.v_ls = p->value_ls; keys.v_ns = token_stride(p->n, p->value_ns, p->o); keys.v_gs = p->value_gs;
    keys.lengths = p->key_lengths;
    keys.mask = p->key_mask; keys.mask_ls = p->key_mask_ls; keys.mask_ns = p->key_mask_ns;
    keys.n = p->n;
    args.grad_q = p->grad_q; args.grad_k = p->grad_key; args.grad_v = p->grad_value;
    args.l = p->l; args.m = p->m; args.g = p->g; args.r = p->h / p->g; args.k = p->k; args.o = p->o;
    args.key_entries = p->key_entries;
    args.scale = p->scale;
    set_scale(p->scale, &args.scale_log2, &args.query_factor);
    args.partial_k_width = (p->k + 3) / 4 * 4;
    args.partial_o_width = (p->o + 3) / 4 * 4;

    const int64_t rows = static_cast<int64_t>(p->m) * args.r;
    args.q_row_tiles = static_cast<int>((rows + 127) / 128);
    const int64_t q_base = static_cast<int64_t>(p->l) * p->g * args.q_row_tiles;
    // a tile of the queries' kernel is 64 keys (32 of rows above 256 bytes), of the keys' kernel 32 rows; two workgroups share a CU where rows have at most
    // 256 bytes (queries) or 128 (keys)
    const double width = padded_width(std::max(p->k, p->o)), slower = p->type == KMC_FP32 ? 7.0 : 1.0;
    const int64_t row_bytes = static_cast<int64_t>(width) * element_size(p->type), q_tile = row_bytes <= 256 ? 64 : 32;
    const double q_elements = static_cast<double>(p->l) * p->m * p->h * p->k, k_elements = static_cast<double>(p->key_entries) * p->n * p->g * (p->k + p->o);
    args.q_splits = may_cut ? parts(q_base, row_bytes <= 256 ? 512 : 256, (p->n + q_tile - 1) / q_tile, 2.4 * width / 128 * slower * (row_bytes <= 256 ? 1.0 : 0.3), q_elements) : 1;
    args.key_tiles = (p->n + 127) / 128;
    const int64_t k_base = static_cast<int64_t>(p->key_entries) * p->g * args.key_tiles;
    const int64_t tiles_of_rows = static_cast<int64_t>(args.r) * ((p->m + 31) / 32) * (p->key_entries == p->l ? 1 : p->l);
    args.k_splits = may_cut ? parts(k_base, row_bytes <= 128 ? 512 : 256, tiles_of_rows, 1.2 * width / 128 * slower * (row_bytes <= 128 ? 1.6 : 1.0), k_elements) : 1;
    const int64_t q_workgroups = q_base * args.q_splits, k_workgroups = k_base * args.k_splits;
    if (std::max(q_workgroups, k_workgroups) > 0x7ffffff0ll) return fail(KMC_ERR_INVALID_ARGUMENT, "more workgroups than the kernels count");
    args.q_workgroups = static_cast<int>(q_workgroups);
    args.q_grid = static_cast<int>((q_workgroups + 7) / 8 * 8);
    args.k_workgroups = static_cast<int>(k_workgroups);
    args.k_grid = static_cast<int>((k_workgroups + 7) / 8 * 8);

    const int64_t q_rows = static_cast<int64_t>(p->l) * p->m * p->h, k_rows = static_cast<int64_t>(p->key_entries) * p->n * p->g;
    plan->stats_bytes = (8 * q_rows + 8 + 15) / 16 * 16;
    plan->shift_bytes = (4 * q_rows + 4 * q_base + 15) / 16 * 16;
    if (args.q_splits > 1) plan->q_bytes = 4ll * args.q_splits * q_rows * args.partial_k_width;
    if (args.k_splits > 1) {
        plan->k_bytes = 4ll * args.k_splits * k_rows * args.partial_k_width;
        plan->v_bytes = 4ll * args.k_splits * k_rows * args.partial_o_width;
    }

    Layout layout{element_size(p->type)};
    layout.operand(p->q, p->k); layout.operand(p->out, p->o); layout.operand(p->grad_out, p->o); layout.operand(p->grad_q, p->k);
    layout.stride(p->l, p->q_ls); layout.tokens(p->m, p->q_ms, p->k); layout.stride(p->h, p->q_hs);
    layout.stride(p->l, p->out_ls); layout.stride(p->m, p->out_ms); layout.stride(p->h, p->out_hs);
    layout.stride(p->l, p->grad_out_ls); layout.tokens(p->m, p->grad_out_ms, p->o); layout.stride(p->h, p->grad_out_hs);
    if (p->n > 0) {
        layout.operand(p->key, p->k); layout.operand(p->value, p->o); layout.operand(p->grad_key, p->k); layout.operand(p->grad_value, p->o);
        layout.stride(p->l, p->key_ls); layout.tokens(p->n, p->key_ns, p->k); layout.stride(p->g, p->key_gs);
        layout.stride(p->l, p->value_ls); layout.tokens(p->n, p->value_ns, p->o); layout.stride(p->g, p->value_gs);
    }
    plan->aligned = layout.aligned && !(p->flags & KMC_FLAG_FORCE_SCALAR_ACCESS);
    return KMC_OK;
}

}  // namespace

extern "C" {

int kmc_attention_workspace_bytes(const kmc_attention_params *params, int64_t *bytes)
{
    if (!bytes) return fail(KMC_ERR_INVALID_ARGUMENT, "bytes: null pointer");
    Plan plan;
    const int status = prepare(params, true, &plan);
    if (status != KMC_OK) return status;
    *bytes = plan.bytes;
    return KMC_OK;
}

int kmc_attention(const kmc_attention_params *params, void *stream)
{
    Plan plan;
    int status = prepare(params, true, &plan);
    if (status != KMC_OK) return status;
    if (plan.empty) return KMC_OK;
    if (plan.bytes > 0 && (!params->workspace || params->workspace_bytes < plan.bytes)) {
        status = prepare(params, false, &plan);
        if (status != KMC_OK) return status;
    }
    status = require_gfx950();
    if (status != KMC_OK) return status;
    kmc::AttentionArgs &args = plan.args;
    if (plan.bytes > 0) {
        if (!aligned16(params->workspace)) return fail(KMC_ERR_INVALID_ARGUMENT, "workspace is not aligned to 16 bytes");
        args.partial_out = static_cast<float *>(params->workspace);
        args.partial_shift = args.partial_out + args.slots * args.rows_total * args.partial_width;
        args.partial_lse = args.partial_shift + args.slots * args.rows_total;
    }
    const int width = std::max(params->k, params->o);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    const hipError_t e = params->type == KMC_FP32   ? launch_attention_forward_0(args, width, plan.aligned, on)
                         : params->type == KMC_FP16 ? launch_attention_forward_1(args, width, plan.aligned, on)
                                                    : launch_attention_forward_2(args, width, plan.aligned, on);
    if (e != hipSuccess) return fail_hip(e, "attention launch");
    return KMC_OK;
}

int kmc_attention_gradient_workspace_bytes(const kmc_attention_gradient_params *params, int64_t *bytes)
{
    if (!bytes) return fail(KMC_ERR_INVALID_ARGUMENT, "bytes: null pointer");
    GradPlan plan;
    const int status = prepare(params, true, &plan);
    if (status != KMC_OK) return status;
    *bytes = plan.bytes();
    return KMC_OK;
}

int kmc_attention_gradient(const kmc_attention_gradient_params *params, void *stream)
{
    GradPlan plan;
    int status = prepare(params, true, &plan);
    if (status != KMC_OK) return status;
    if (plan.empty) return KMC_OK;
    if (!params->workspace || params->workspace_bytes < plan.bytes()) {
        status = prepare(params, false, &plan);
        if (status != KMC_OK) return status;
        if (params->workspace_bytes < plan.bytes()) plan.shift_bytes = 0;
        if (!params->workspace || params->workspace_bytes < plan.bytes())
            return fail(KMC_ERR_INVALID_ARGUMENT, "the gradient of attention needs a workspace of %lld bytes", static_cast<long long>(plan.bytes()));
    }
    if (!aligned16(params->workspace)) return fail(KMC_ERR_INVALID_ARGUMENT, "workspace is not aligned to 16 bytes");
    status = require_gfx950();
    if (status != KMC_OK) return status;
    kmc::AttentionGradArgs &args = plan.args;
    char *at = static_cast<char *>(params->workspace);
    args.stats = reinterpret_cast<float *>(at);
    at += plan.stats_bytes;
    if (plan.shift_bytes > 0) {
        args.row_shift = reinterpret_cast<float *>(at);
        args.row_flags = reinterpret_cast<int *>(at) + static_cast<int64_t>(args.l) * args.m * args.g * args.r;
    }
    args.partial_q = reinterpret_cast<float *>(at += plan.shift_bytes);
    args.partial_k = reinterpret_cast<float *>(at += plan.q_bytes);
    args.partial_v = reinterpret_cast<float *>(at += plan.k_bytes);
    const int width = std::max(params->k, params->o);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    const hipError_t e = params->type == KMC_FP32   ? launch_attention_gradient_0(args, width, plan.aligned, on)
                         : params->type == KMC_FP16 ? launch_attention_gradient_1(args, width, plan.aligned, on)
                                                    : launch_attention_gradient_2(args, width, plan.aligned, on);
    if (e != hipSuccess) return fail_hip(e, "attention gradient launch");
    return KMC_OK;
}

}  // extern "C"
