// Byte offsets within a row of an operand, in 64 bits: a row has up to 2^31 - 2^16 values, its bytes pass 32 bits from 2^29 pairs
// and from 2^30 half-precision values on.  Nothing here needs the GPU compiler.
#ifndef ODAMD_OFFSETS_H
#define ODAMD_OFFSETS_H

// Value k's hi within a row of pairs (32 hi, then their 32 lo); its lo lies 64 bytes on.
constexpr long long split_at(int k) { return (long long)(k >> 5) * 128 + (k & 31) * 2; }
// Columns col .. col + 7 of a row of `cols` half-precision values, col a multiple of eight; columns past the last as the last eight.
constexpr long long column_at(int col, int cols) {
    const int last = (cols - 1) & ~7;
    return (long long)(col < last ? col : last) * 2;
}

#endif
