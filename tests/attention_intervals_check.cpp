// Compares the two sides of the relation "row i sees key j" with its definition, over all small sizes and at the largest ones.
#include <algorithm>
#include <cstdio>
#include "../sddmm_gpu_amd/csrc/attention_intervals.hpp"

using namespace sddmm;

// max(0, pos - left) <= j < min(n_k, max(pos + right + 1, prefix)), in 64 bits; windows of -1 have no bound
static bool sees(int64_t n_q, int64_t n_k, int64_t left, int64_t right, int64_t prefix, int64_t i, int64_t j)
{
    const int64_t pos = n_k - n_q + i;
    const int64_t lo = left < 0 ? 0 : std::max<int64_t>(0, pos - left), hi = right < 0 ? n_k : std::min(n_k, std::max(pos + right + 1, prefix));
    return lo <= j && j < hi;
}

static long bad = 0;
static void check(int n_q, int n_k, int left, int right, int prefix, int i, int j)
{
    const int shift = n_k - n_q, pos = i + shift;
    const bool want = sees(n_q, n_k, left, right, prefix, i, j);
    const bool of_row = first_key(left, pos) <= j && j < end_key(right, pos, prefix, n_k);
    const bool of_key = first_row(right, j, prefix, shift) <= i && i < end_row(left, j, shift, n_q);
    if ((of_row != want || of_key != want) && bad++ < 5)
        printf("n_q %d n_k %d left %d right %d prefix %d row %d key %d: %d, by the row %d, by the key %d\n", n_q, n_k, left, right, prefix, i, j, want, of_row, of_key);
}

int main()
{
    for (int n_q = 0; n_q <= 9; ++n_q)
        for (int n_k = 0; n_k <= 9; ++n_k)
            for (int left = -1; left <= 12; ++left)
                for (int right = -1; right <= 12; ++right)
                    for (int prefix = -1; prefix <= 11; ++prefix)
                        for (int i = 0; i < n_q; ++i)
                            for (int j = 0; j < n_k; ++j) check(n_q, n_k, left, right, prefix, i, j);
    const int most = INT32_MAX / 2, sizes[] = {1, 2, 77, most - 1, most}, windows[] = {-1, 0, 1, 50, most, 1 << 30};
    for (int n_q : sizes)
        for (int n_k : sizes)
            for (int left : windows)
                for (int right : windows)
                    for (int prefix : {0, 1, n_k, INT32_MAX})
                        for (int i : {0, 1, n_q / 2, n_q - 2, n_q - 1})
                            for (int j : {0, 1, n_k / 2, n_k - 2, n_k - 1})
                                if (i >= 0 && i < n_q && j >= 0 && j < n_k) check(n_q, n_k, left, right, prefix, i, j);
    printf("%ld differ\n", bad);
    return bad != 0;
}
