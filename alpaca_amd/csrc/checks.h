// Argument checks and the launch's status, shared by the entry points that take device
// pointers and a stream.
#pragma once

#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/alpaca_hip.h"
#include "host.h"

// ahip_fail, which no exception leaves.
inline int failed(int code, const char* text) {
    try {
        return ahip_fail(code, text);
    } catch (...) {
        return code;
    }
}

// AHIP_ERR_INVALID_ARGUMENT with a message, printf's way; without host memory, with none.
__attribute__((format(printf, 1, 2))) inline int bad(const char* format, ...) {
    char text[256];
    va_list args;
    va_start(args, format);
    vsnprintf(text, sizeof(text), format, args);
    va_end(args);
    return failed(AHIP_ERR_INVALID_ARGUMENT, text);
}

inline int launched(hipError_t e) {
    if (e == hipSuccess) return AHIP_OK;
    (void)hipGetLastError();
    char text[256];
    snprintf(text, sizeof(text), "kernel launch: %s", hipGetErrorString(e));
    return failed(AHIP_ERR_COMMAND_FAILED, text);
}

inline int check_dim(int hd) {
    if (hd <= 0 || hd % 32 || hd > 256) return bad("head dimension must be a multiple of 32 up to 256");
    return AHIP_OK;
}

inline int check_dtype(int dtype) {
    if (dtype != AHIP_F32 && dtype != AHIP_F16) return bad("rows must be f32 or f16");
    return AHIP_OK;
}

// Rows of `width` elements, `stride` elements apart.
inline int check_rows(const char* what, const void* p, int64_t stride, int64_t width, int dtype) {
    if (!p) return bad("null %s", what);
    if ((uintptr_t)p % (dtype == AHIP_F32 ? 4 : 2)) return bad("%s: misaligned", what);
    if (stride < width) return bad("%s: stride below the row's width", what);
    if (stride > (int64_t)1 << 32) return bad("%s: implausibly large stride", what);
    return AHIP_OK;
}

inline int stream_of(ahip_context* ctx, ahip_stream* stream, hipStream_t* out) {
    if (stream && stream->device != ctx->device) return bad("stream and context belong to different devices");
    (void)hipGetLastError();  // a launch's own failure is read back through it
    if (hipSetDevice(ctx->device) != hipSuccess) return failed(AHIP_ERR_COMMAND_FAILED, "hipSetDevice");
    *out = stream ? stream->st : ctx->stream;
    return AHIP_OK;
}
