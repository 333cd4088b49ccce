// Operators that treat a row (a pixel's channels) of a channels-last map as one vector: root-mean-square normalisation, 8-bit
// codes with a scale per row, the pointwise convolution of those, and counter-based dropout. Shared host definitions.
#pragma once

#include "maps.h"

namespace tvdcn_hip {

// ---- launchers (rms_norm.hip, pointwise_int8.hip, dropout.hip): asynchronous on `s`, nothing allocated ----

struct RowArgs {
    int dtype;
    int64_t rows;
    int channels;
    float eps;
    const void *x, *residual;     // residual: or null
    const void *weight;           // [channels] or null
    void *sum;                    // x + residual in the map's type, where there is a residual
    void *y;
    float *rstd;                  // [rows], or null where no backward follows
    int8_t *codes;
    float *scales;                // [rows]
};
hipError_t launch_rms_norm(const RowArgs &a, hipStream_t s);
hipError_t launch_rms_norm_int8(const RowArgs &a, hipStream_t s);
hipError_t launch_quantize(const RowArgs &a, hipStream_t s);
hipError_t launch_dequantize(int dtype, int64_t rows, int channels, const int8_t *codes, const float *scales, void *y, hipStream_t s);

struct RowGradArgs {
    int dtype;
    int64_t rows;
    int channels;
    const void *dy, *dsum;        // gradients of both results (dsum: or null)
    const void *x;                // what was normalised
    const float *rstd;
    const void *weight;
    void *dx, *dweight;           // null: not asked for
    float *part;                  // workspace
};
int64_t rms_norm_part_floats(const RowGradArgs &a);
hipError_t launch_rms_norm_backward(const RowGradArgs &a, hipStream_t s);

struct Int8ProductArgs {
    int dtype, act;               // of y
    int64_t rows;
    int in, out;
    const int8_t *codes, *weight_codes;
    const float *scales, *weight_scales;
    const void *bias, *residual;
    void *y;
    char *work;
};
size_t pointwise_int8_bytes(const Int8ProductArgs &a);
hipError_t launch_pointwise_int8(const Int8ProductArgs &a, hipStream_t s);

// drop: values are dropped where their 16 bits are below it
hipError_t launch_dropout(int dtype, int64_t n, int drop, const int64_t *seed, const void *x, const void *residual, void *y,
                          hipStream_t s);

}  // namespace tvdcn_hip
