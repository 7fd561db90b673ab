// Sums over a wave's lanes and values of single lanes, of 32 or 64 bits, by VALU moves (a
// shuffle through the LDS crossbar takes several times as long).  All lanes take part.
#pragma once
#include "qg_common.h"

// A value of another lane by a VALU move, 0 where there is none or the row is not in ROWS; in 32-bit words.
template <int CTRL, int ROWS, typename T>
QG_DEV T moved_lane(T v) {
    if constexpr (sizeof(T) == 8) {
        const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(T, (unsigned long long)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    }
}
// Sums over the lanes up to each: within rows of 16, then the rows' last lanes to those behind.
template <typename T>
QG_DEV T wave_upto(T v) {
    v += moved_lane<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
    v += moved_lane<0x112, 0xf>(v);
    v += moved_lane<0x114, 0xf>(v);
    v += moved_lane<0x118, 0xf>(v);
    v += moved_lane<0x142, 0xa>(v);  // row_bcast 15, 31
    v += moved_lane<0x143, 0xc>(v);
    return v;
}
// The value of a lane that all lanes name.
template <typename T>
QG_DEV T of_lane(T v, int l) {
    if constexpr (sizeof(T) == 8) {
        const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l);
        return __builtin_bit_cast(T, (unsigned long long)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
    }
}
template <typename T>
QG_DEV T wave_all_add(T v) { return of_lane(wave_upto(v), 63); }
