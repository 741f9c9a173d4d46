// Rotary positions of queries and keys (gfx950).
#include <hip/hip_runtime.h>
#include <cmath>
#include <cstring>
#include "internal.hpp"
#include "launch.hpp"

using namespace sddmm;

namespace {

constexpr int kBlock = 256;
constexpr int kTable = 1024;  // pairs whose cosine and sine a workgroup holds

struct RotaryArgs {
    const int32_t *positions;
    const double *freq;
    const void *x[2];   // q and k
    void *y[2];
    int64_t x_row[2], x_head[2], y_row[2], y_head[2];
    int64_t n_rows, first_position;
    int32_t heads[2], head_dim, rot_dim, per_row, copy;  // per_row: rows of a workgroup; copy: the rest of a head is copied
    float amplitude, sign;
};

template <class T, int N> struct Piece { typedef T Vec __attribute__((ext_vector_type(N))); };
template <class T> struct Piece<T, 1> { typedef T Vec; };

// cos and sin of 2 pi t, |t| <= 1/8: the series up to the terms below 2^-25 of the result
__device__ __forceinline__ void near_zero(float t, float &c, float &s)
{
    const float x = t * 6.283185307179586f, z = x * x;
    s = x * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -0.16666667f), 1.f);
    c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
}

// One pass at copy speed is the aim: the angles' cosines and sines are made once for all heads of a row and kept in LDS (per pair 2
// double-precision products and about 25 instructions; made anew for each head they would take as long as the copy), then every thread turns pieces of
// V elements (16 bytes where sizes and alignment allow it) of the heads of q and k in one launch.  The angle in turns is reduced in
// 64 bits: at position 10^6 a 32-bit product would be off by 0.06 radians.  Results are rounded once.
// 16,384 rows of 32 + 8 heads of 128, 96 elements turned, interleaved, bf16: 60 us = 5.6 TB/s read and written (a large copy 5.0); 64 rows 4.4 us.
template <class T, int V, bool HALF>
__global__ __launch_bounds__(kBlock)
void sddmm_rotary_kernel(const RotaryArgs a)
{
    typedef typename Piece<T, V>::Vec Vec;
    constexpr int kPairs = V > 1 ? V / 2 : 1;  // of a piece, where pairs are neighbours
    __shared__ float2 table[kTable];
    const int pairs = a.rot_dim / 2;
    const int64_t row0 = (int64_t)blockIdx.x * a.per_row;
    const int rows = (int)min((int64_t)a.per_row, a.n_rows - row0);
    // Pairs beyond the table are turned in further rounds; the last one also copies the rest of the heads, whose lines the pairs' pieces lie in.
    for (int p0 = 0; p0 < pairs; p0 += kTable) {
        const int some = min(pairs - p0, kTable);
        if (p0) __syncthreads();
        for (int i = threadIdx.x; i < rows * some; i += kBlock) {
            const int r = i / some, p = i - r * some;
            const double pos = a.positions ? (double)a.positions[row0 + r] : (double)(a.first_position + row0 + r);
            const double turns = pos * (a.freq[p0 + p] * 0.15915494309189533577);
            const double part = turns - rint(turns);
            const double quarter = rint(part * 4.);
            float c, s;
            near_zero((float)(part - quarter * 0.25), c, s);
            const int k = (int)quarter & 3;
            const float cosine = k == 0 ? c : k == 1 ? -s : k == 2 ? -c : s, sine = k == 0 ? s : k == 1 ? c : k == 2 ? -s : -c;
            table[i] = make_float2(cosine * a.amplitude, sine * a.amplitude * a.sign);
        }
        __syncthreads();
        // Two pieces of a head to a thread where that is possible: the two of pairs in halves, or one and the one half of all pieces on; pieces that are copied likewise
        // (us, 16,384 rows of 32 + 8 heads of 128, 96 of them turned, interleaved, one and two pieces 78 and 64, 2048 rows 10.1 and 8.4).
        const int turned = some / (HALF ? V : kPairs), copied = a.copy && p0 + some == pairs ? (a.head_dim - a.rot_dim) / V : 0;
        const bool two = V > 1 && (HALF ? copied : turned + copied) % 2 == 0;
        const int items = HALF ? turned + (two ? copied / 2 : copied) : two ? (turned + copied) / 2 : turned + copied;
        const int all_heads = a.heads[0] + a.heads[1], n = rows * all_heads * items;
        const float by_items = 1.f / (float)items, by_heads = 1.f / (float)all_heads;
        for (int i = threadIdx.x; i < n; i += kBlock) {
            // (quotients by a product: exact below 2^20, which n is held to)
            const int unit = (int)(((float)i + 0.5f) * by_items), item = i - unit * items;
            const int r = (int)(((float)unit + 0.5f) * by_heads), head_at = unit - r * all_heads;
            const int which = head_at >= a.heads[0], head = which ? head_at - a.heads[0] : head_at;
            const T *x = (const T *)a.x[which] + (row0 + r) * a.x_row[which] + head * a.x_head[which];
            T *y = (T *)a.y[which] + (row0 + r) * a.y_row[which] + head * a.y_head[which];
            const float2 *angles = &table[r * some];
            if constexpr (HALF || V == 1) {
                // (items to turn and to copy lie in one wave: loads and stores are common to both)
                const bool turn = item < turned, both = turn || two;
                const int at = !turn ? a.rot_dim + (item - turned) * V : HALF ? p0 + item * V : 2 * (p0 + item);
                const int other = !turn ? (two ? at + copied / 2 * V : at) : HALF ? at + pairs : at + 1;
                Vec u = *(const Vec *)(x + at), v = *(const Vec *)(x + other);
                if (turn) {
                    const float2 *cs = angles + item * V;
                    if constexpr (V == 1) {
                        const float f = (float)u, g = (float)v;
                        u = (T)(f * cs[0].x - g * cs[0].y), v = (T)(f * cs[0].y + g * cs[0].x);
                    } else {
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const float f = (float)u[j], g = (float)v[j];
                            u[j] = (T)(f * cs[j].x - g * cs[j].y), v[j] = (T)(f * cs[j].y + g * cs[j].x);
                        }
                    }
                }
                *(Vec *)(y + at) = u;
                if (both) *(Vec *)(y + other) = v;
            } else {
                auto place = [&](int k) { return k < turned ? 2 * p0 + k * V : a.rot_dim + (k - turned) * V; };
                auto turn = [&](Vec &u, int k) {
                    if (k >= turned) return;
                    const float2 *cs = angles + k * kPairs;
#pragma unroll
                    for (int j = 0; j < kPairs; ++j) {
                        const float f = (float)u[2 * j], g = (float)u[2 * j + 1];
                        u[2 * j] = (T)(f * cs[j].x - g * cs[j].y), u[2 * j + 1] = (T)(f * cs[j].y + g * cs[j].x);
                    }
                };
                Vec u = *(const Vec *)(x + place(item)), v = u;
                if (two) v = *(const Vec *)(x + place(item + items));
                turn(u, item);
                *(Vec *)(y + place(item)) = u;
                if (two) {
                    turn(v, item + items);
                    *(Vec *)(y + place(item + items)) = v;
                }
            }
        }
    }
}

template <class T>
hipError_t launch_typed(const RotaryArgs &a, int v, bool half, hipStream_t st)
{
    void (*fn)(RotaryArgs) = nullptr;
    if constexpr (sizeof(T) == 2) {
        if (v == 8) fn = half ? sddmm_rotary_kernel<T, 8, true> : sddmm_rotary_kernel<T, 8, false>;
    }
    if (!fn) fn = v >= 4 ? (half ? sddmm_rotary_kernel<T, 4, true> : sddmm_rotary_kernel<T, 4, false>)
                : v == 2 ? (half ? sddmm_rotary_kernel<T, 2, true> : sddmm_rotary_kernel<T, 2, false>)
                : (half ? sddmm_rotary_kernel<T, 1, true> : sddmm_rotary_kernel<T, 1, false>);
    return launch(fn, dim3((unsigned)((a.n_rows + a.per_row - 1) / a.per_row)), dim3(kBlock), 0, st, a);
}

}  // namespace

extern "C" {

void sddmm_rotary_desc_init(sddmm_rotary_desc *desc)
{
    if (!desc) return;
    memset(desc, 0, sizeof *desc);
    desc->amplitude = 1.f;
}

int sddmm_rotary(const sddmm_rotary_desc *desc, const int32_t *d_positions, const double *d_freq, const void *d_q, void *d_q_out,
                 const void *d_k, void *d_k_out, void *stream)
{
    const char *who = "sddmm_rotary";
    if (!desc) return fail(SDDMM_ERR_ARG, "%s: NULL description", who);
    const sddmm_rotary_desc &d = *desc;
    if (d.type != SDDMM_TYPE_F32 && d.type != SDDMM_TYPE_BF16 && d.type != SDDMM_TYPE_F16) return fail(SDDMM_ERR_ARG, "%s: unknown type %d", who, d.type);
    if (d.layout != SDDMM_ROTARY_HALF && d.layout != SDDMM_ROTARY_INTERLEAVED) return fail(SDDMM_ERR_ARG, "%s: unknown layout %d", who, d.layout);
    if (d.head_dim < 2 || d.head_dim > 4096 || d.rot_dim < 2 || d.rot_dim % 2 || d.rot_dim > d.head_dim)
        return fail(SDDMM_ERR_ARG, "%s: rot_dim = %d has to be even and 2 .. head_dim = %d, which is up to 4096", who, d.rot_dim, d.head_dim);
    if (d.n_heads < 1 || d.n_kv_heads < 0 || d.n_rows < 0) return fail(SDDMM_ERR_ARG, "%s: no heads, or a negative size", who);
    if (!std::isfinite(d.amplitude)) return fail(SDDMM_ERR_ARG, "%s: amplitude must be finite", who);
    const bool keys = d.n_kv_heads > 0;
    const int64_t strides[2][4] = {{d.q_row, d.q_head, d.q_out_row, d.q_out_head}, {d.k_row, d.k_head, d.k_out_row, d.k_out_head}};
    const int32_t heads[2] = {d.n_heads, d.n_kv_heads};
    for (int w = 0; w <= (keys ? 1 : 0); ++w)
        for (int i = 0; i < 4; ++i)
            if (strides[w][i] < 0 || ((i % 2 ? heads[w] > 1 : d.n_rows > 1) && strides[w][i] < d.head_dim)) return fail(SDDMM_ERR_ARG, "%s: a stride below head_dim", who);
    // rows and heads that lie in each other's place would be written twice
    for (int w = 0; w <= (keys ? 1 : 0); ++w) {
        const int64_t row = strides[w][2], head = strides[w][3];
        if (d.n_rows > 1 && heads[w] > 1 && row < (heads[w] - 1) * head + d.head_dim && head < (d.n_rows - 1) * row + d.head_dim)
            return fail(SDDMM_ERR_ARG, "%s: rows and heads of the results overlap", who);
    }
    if (d.n_rows > ((int64_t)1 << 40) || (int64_t)d.n_heads + d.n_kv_heads > 65536) return fail(SDDMM_ERR_RANGE, "%s: too many rows or heads", who);
    if (d.n_rows == 0) return SDDMM_OK;
    if (!d_freq || !d_q || !d_q_out || (keys && (!d_k || !d_k_out))) return fail(SDDMM_ERR_ARG, "%s: NULL device pointer", who);
    const int size = d.type == SDDMM_TYPE_F32 ? 4 : 2;
    uint64_t low = (uintptr_t)d_q | (uintptr_t)d_q_out | (keys ? (uintptr_t)d_k | (uintptr_t)d_k_out : 0);
    if (low % size || (uintptr_t)d_freq % 8 || (uintptr_t)d_positions % 4) return fail(SDDMM_ERR_ARG, "%s: pointers must be aligned to their elements", who);
    // (threads of the same and of other workgroups still read what a result in any other place would overwrite)
    auto moved = [&](int w) { return (d.n_rows > 1 && strides[w][0] != strides[w][2]) || (heads[w] > 1 && strides[w][1] != strides[w][3]); };
    if ((d_q == d_q_out && moved(0)) || (keys && ((d_k == d_k_out && moved(1)) || d_q_out == d_k || d_k_out == d_q || d_q_out == d_k_out)))
        return fail(SDDMM_ERR_ARG, "%s: a result is in an operand's or the other result's place (only its own operand's, with the same strides, is taken)", who);

    RotaryArgs a{};
    a.positions = d_positions, a.freq = d_freq;
    a.x[0] = d_q, a.y[0] = d_q_out, a.x[1] = d_k, a.y[1] = d_k_out;
    for (int w = 0; w < 2; ++w) {
        a.heads[w] = heads[w];
        a.x_row[w] = strides[w][0], a.x_head[w] = strides[w][1], a.y_row[w] = strides[w][2], a.y_head[w] = strides[w][3];
    }
    a.n_rows = d.n_rows, a.first_position = d.first_position, a.head_dim = d.head_dim, a.rot_dim = d.rot_dim;
    a.amplitude = d.amplitude, a.sign = d.inverse ? -1.f : 1.f;
    const bool in_place = d_q == d_q_out && d.q_row == d.q_out_row && d.q_head == d.q_out_head &&
                          (!keys || (d_k == d_k_out && d.k_row == d.k_out_row && d.k_head == d.k_out_head));
    a.copy = d.rot_dim < d.head_dim && !in_place;
    // the widest piece that all offsets are multiples of
    uint64_t bits = low / size;
    for (int w = 0; w <= (keys ? 1 : 0); ++w)
        for (int i = 0; i < 4; ++i) bits |= (uint64_t)strides[w][i];
    bits |= (uint64_t)(d.layout == SDDMM_ROTARY_HALF ? d.rot_dim / 2 : d.rot_dim);
    if (a.copy) bits |= (uint64_t)(d.head_dim - d.rot_dim);
    int v = 16 / size;
    while (v > 1 && bits % v) v /= 2;
    const bool half = d.layout == SDDMM_ROTARY_HALF;
    // Rows of a workgroup: as many as have one and a half pairs of pieces for each thread, but 1024 workgroups (us, 16,384 rows of 32 + 8 heads of 128, interleaved, one and two
    // rows 61 and 64; of 8 + 2 heads one, two, four, five and six 28, 21, 18, 17 and 17; of 2 + 2 heads of 64, in halves 14, 9 and, with twelve, 7.5).
    const int64_t pieces = d.rot_dim / (half || v == 1 ? 2 * v : v) + (d.head_dim - d.rot_dim) / v + 1, row_work = pieces * (d.n_heads + d.n_kv_heads);
    if (row_work > (1 << 20)) return fail(SDDMM_ERR_RANGE, "%s: a row of all heads is too long", who);
    a.per_row = (int)std::max<int64_t>(1, std::min<int64_t>({d.n_rows / 1024, (int64_t)kTable / (d.rot_dim / 2), ((int64_t)1 << 20) / row_work, 384 / std::max<int64_t>(1, row_work / 2)}));
    const int64_t grid = (d.n_rows + a.per_row - 1) / a.per_row;
    if (!launchable(grid, kBlock)) return fail(SDDMM_ERR_RANGE, "%s: too many rows for one launch", who);
    const hipStream_t st = (hipStream_t)stream;
    const hipError_t e = d.type == SDDMM_TYPE_F32 ? launch_typed<float>(a, v, half, st) : d.type == SDDMM_TYPE_F16 ? launch_typed<_Float16>(a, v, half, st)
                                                                                                                 : launch_typed<__bf16>(a, v, half, st);
    if (e != hipSuccess) return fail(SDDMM_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
    return SDDMM_OK;
}

int sddmm_rotary_frequencies(int32_t rot_dim, double base, int32_t scaling, double factor, int64_t known_len, double low, double high,
                             double *freq, double *amplitude)
{
    const char *who = "sddmm_rotary_frequencies";
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > 4096) return fail(SDDMM_ERR_ARG, "%s: rot_dim = %d has to be even and 2 .. 4096", who, rot_dim);
    if (!(base > 1.) || !std::isfinite(base)) return fail(SDDMM_ERR_ARG, "%s: base must be above 1", who);
    if (scaling < SDDMM_ROTARY_PLAIN || scaling > SDDMM_ROTARY_PARTS) return fail(SDDMM_ERR_ARG, "%s: unknown scaling %d", who, scaling);
    if (!freq || !amplitude) return fail(SDDMM_ERR_ARG, "%s: NULL pointer", who);
    if (scaling != SDDMM_ROTARY_PLAIN && (!(factor >= 1.) || !std::isfinite(factor))) return fail(SDDMM_ERR_ARG, "%s: factor must be 1 or more", who);
    const bool turns = scaling == SDDMM_ROTARY_BANDS || scaling == SDDMM_ROTARY_PARTS;
    if (turns && (known_len < 1 || !(low > 0.) || !(high > low) || !std::isfinite(high)))
        return fail(SDDMM_ERR_ARG, "%s: known_len has to be 1 or more and 0 < low < high", who);
    const double pi2 = 6.283185307179586477;
    if (scaling == SDDMM_ROTARY_BASE) base *= std::pow(factor, rot_dim / std::max(1., rot_dim - 2.));
    *amplitude = scaling == SDDMM_ROTARY_PARTS ? 0.1 * std::log(factor) + 1. : 1.;
    // (the pair that makes so many turns in known_len)
    auto pair = [&](double t) { return rot_dim * std::log(known_len / (t * pi2)) / (2. * std::log(base)); };
    const double from = turns ? std::max(0., std::floor(pair(high))) : 0., to = turns ? std::min(rot_dim - 1., std::ceil(pair(low))) : 0.;
    for (int e = 0; e < rot_dim / 2; ++e) {
        double f = std::pow(base, -2. * e / rot_dim), keep = 1.;
        if (scaling == SDDMM_ROTARY_LINEAR) keep = 0.;
        if (scaling == SDDMM_ROTARY_BANDS) keep = std::min(1., std::max(0., (known_len * f / pi2 - low) / (high - low)));
        if (scaling == SDDMM_ROTARY_PARTS) keep = 1. - std::min(1., std::max(0., (e - from) / std::max(to - from, 0.001)));
        freq[e] = f * (keep + (1. - keep) / factor);
    }
    return SDDMM_OK;
}

}  // extern "C"
