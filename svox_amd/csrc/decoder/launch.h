// launch.h -- what the units of a library of operators share on the host: errors, launches of any size, a caller's workspace.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace svox_decoder {

// (defined by each library)
__attribute__((format(printf, 2, 3))) int fail(int code, const char* fmt, ...);
int check_launch(const char* what);

// `blocks` blocks of a launch.  The runtime counts a launch's threads along each axis in 32 bits and runs what is left of a larger number,
// without an error (of the 16 777 218 blocks of 256 that 2^30 + 77 rows came to it ran two): such a launch gets no blocks here, which is
// an error that check_launch sees.
inline dim3 grid_of(int64_t blocks, int threads) { return dim3(blocks < ((int64_t)1 << 32) / threads ? (unsigned)blocks : 0); }

// A caller's workspace, given out in pieces of whole 256 bytes; with no address, only counted.
struct Room {
    char* at;
    int64_t used = 0;
    explicit Room(void* base) : at((char*)base) {}
    template <class T>
    T* take(int64_t count) {
        T* const p = at ? (T*)(at + used) : nullptr;
        used += (count * (int64_t)sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

}  // namespace svox_decoder
