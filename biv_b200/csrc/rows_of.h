// A request's rows from a list of offsets.  Plain C++, without the CUDA headers, so that it can be tested where there is no GPU.
#pragma once

#ifdef __CUDACC__
#define BIV_ROWS_FN __host__ __device__ __forceinline__
#else
#define BIV_ROWS_FN inline
#endif

namespace bivmoe {

struct RowsOf { int first, n; };
// Both offsets are kept within 0..n_tokens before their difference is taken, which whatever stands in the list does not overflow then:
// of -2^31 behind 130 it was 2^31 - 130 rows.
BIV_ROWS_FN RowsOf rows_of(int from, int to, int n_tokens) {
    const int a = from < 0 ? 0 : from < n_tokens ? from : n_tokens, b = to < 0 ? 0 : to < n_tokens ? to : n_tokens;
    return RowsOf{a, b > a ? b - a : 0};
}

}  // namespace bivmoe
