// How a piece of eight elements of 16 bits that starts anywhere is read (ldn_gated.cu): by itself, so that the ranges can be checked on the
// host.
#pragma once
#ifdef __CUDACC__
#define LDN_BOTH __host__ __device__ __forceinline__
#else
#define LDN_BOTH inline
#endif

namespace ldn {

// 1: as one aligned word of 16 bytes, 2: from the two aligned words that it lies in, 0: element by element.  off: its place in 16 bytes; c: its
// column, a multiple of eight.  Both words are the tensor's where they lie in the row, or where other rows lie in front of and behind it: those
// of rows that are repeated (pitch 0) or overlap do not.
LDN_BOTH int words_of_piece(unsigned off, int c, int C, long long row, long long rows, long long pitch) {
    if (c + 8 > C) return 0;
    if (off == 0) return 1;
    const bool apart = pitch >= C;
    return (c > 0 || (apart && row > 0)) && (c + 16 <= C || (apart && row + 1 < rows)) ? 2 : 0;
}

}  // namespace ldn
