// Dense attention: which keys a row sees, and which rows see a key -- one relation from its two sides, both an interval.  Nothing of HIP in it, so that
// the two can be held against each other on a CPU.
//
// pos = row + shift, shift = n_keys - n_rows, which is below 0 where there are more rows than keys: then a row before the first key may see some of them,
// as far as `right` reaches.  Rows and keys are below 2^30 and windows at most 2^30 (or below 0: no bound), so that nothing here passes 32 bits.
#pragma once
#include <cstdint>

namespace sddmm {

// The keys that a row at position pos sees: [first_key, end_key).
constexpr int first_key(int left, int pos) { return left < 0 || pos < left ? 0 : pos - left; }
constexpr int end_key(int right, int pos, int prefix, int n_keys)
{
    if (right < 0) return n_keys;
    const int reach = (pos < INT32_MAX - 1 - right ? pos : INT32_MAX - 1 - right) + right + 1, most = reach > prefix ? reach : prefix;
    return most < n_keys ? most : n_keys;
}

// The rows that see key j: [first_row, end_row).
constexpr int first_row(int right, int j, int prefix, int shift)
{
    const int row = j - right - shift;
    return right < 0 || j < prefix || row < 0 ? 0 : row;
}
constexpr int end_row(int left, int j, int shift, int n_rows)
{
    if (left < 0) return n_rows;
    const int row = j - shift + left + 1;
    return row < 0 ? 0 : row < n_rows ? row : n_rows;
}

}  // namespace sddmm
