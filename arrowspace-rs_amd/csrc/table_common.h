// table_common.h -- what the operators over a table of rows share (table_loss.hip, table4.hip): element types, the checks of
// their entry points, workspaces that a caller may bring.
#pragma once

#include <new>

#include "common.h"

namespace asx {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

inline size_t dtype_size(int dt) { return dt == AS_F64 ? 8 : dt == AS_F32 ? 4 : 2; }
inline bool dtype_is_training(int dt) { return dt == AS_F32 || dt == AS_BF16 || dt == AS_F16; }

// The caller's current device, put back when the call returns: these entry points run inside programs that keep one of their own.
struct DeviceScope {
  int before = -1;
  DeviceScope() {
    if (hipGetDevice(&before) != hipSuccess) before = -1;
  }
  ~DeviceScope() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

// Where a pointer lives: 0 host, 1 the context's device, -1 another device (its kernels cannot be ordered with this context's stream).
inline int pointer_home(as_ctx *ctx, const void *p) {
  hipPointerAttribute_t a;
  if (hipPointerGetAttributes(&a, p) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  if (a.type == hipMemoryTypeManaged) return 1;
  if (a.type != hipMemoryTypeDevice) return 0;
  return a.device == ctx->device ? 1 : -1;
}

// Scratch of one call: the caller's workspace (what a captured graph needs: its addresses stay the graph's own), else blocks of
// the context's cache, which are in use until the call's work on the stream is done and so never part of a graph.
struct Scratch {
  as_ctx *ctx = nullptr;
  char *base = nullptr;
  uint64_t size = 0, used = 0;
  DevBuf<char> own;
  int open(as_ctx *c, void *workspace, uint64_t bytes, uint64_t need) {
    ctx = c;
    size = need;
    if (workspace) {
      if (bytes < need) return fail(c, AS_ERR_ARG, "workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed");
      if ((uintptr_t)workspace & 255) return fail(c, AS_ERR_ARG, "workspace must be aligned to 256 bytes");
      if (need && pointer_home(c, workspace) != 1) return fail(c, AS_ERR_ARG, "workspace must be memory of the context's device");
      base = (char *)workspace;
      return AS_OK;
    }
    if (!need) return AS_OK;
    if (stream_is_capturing(c->stream)) return fail(c, AS_ERR_UNSUPPORTED, "a call on a stream that is being captured needs a workspace of its own");
    AS_TRY(own.alloc(c, need));
    base = own.p;
    return AS_OK;
  }
};

// Sizes of a call's pieces of scratch, taken in the same order for the size and for the addresses.
struct Layout {
  char *base = nullptr;
  uint64_t at = 0;
  template <class T>
  T *take(uint64_t count) {
    T *p = base ? (T *)(base + at) : nullptr;
    at += (count * sizeof(T) + 255) & ~(uint64_t)255;
    return p;
  }
};

// Inputs and outputs of any element type that may live on the host (DevIn / DevOut move whole arrays of one type): staged as bytes.
struct BytesIn {
  const void *p = nullptr;
  DevBuf<char> tmp;
  int bind(as_ctx *ctx, const void *src, uint64_t bytes) {
    p = src;
    if (!src || !bytes) return AS_OK;
    const int home = pointer_home(ctx, src);
    if (home < 0) return fail(ctx, AS_ERR_ARG, "a tensor of another device than the context's");
    if (home == 1) return AS_OK;
    if (stream_is_capturing(ctx->stream)) return fail(ctx, AS_ERR_UNSUPPORTED, "host memory in a call on a stream that is being captured");
    AS_TRY(tmp.alloc(ctx, bytes));
    AS_HIP(ctx, copy_h2d(ctx, tmp.p, src, bytes));
    p = tmp.p;
    return AS_OK;
  }
};
struct BytesOut {
  void *p = nullptr, *host = nullptr;
  uint64_t n = 0;
  DevBuf<char> tmp;
  int bind(as_ctx *ctx, void *dst, uint64_t bytes) {
    p = dst;
    if (!dst || !bytes) return AS_OK;
    const int home = pointer_home(ctx, dst);
    if (home < 0) return fail(ctx, AS_ERR_ARG, "a tensor of another device than the context's");
    if (home == 1) return AS_OK;
    if (stream_is_capturing(ctx->stream)) return fail(ctx, AS_ERR_UNSUPPORTED, "host memory in a call on a stream that is being captured");
    host = dst;
    n = bytes;
    AS_TRY(tmp.alloc(ctx, bytes));
    p = tmp.p;
    return AS_OK;
  }
  int finish(as_ctx *ctx) {
    if (host) AS_HIP(ctx, copy_d2h(ctx, host, p, n));
    return AS_OK;
  }
};
// the same promise as DevOut::finish: on its private stream a context's call is complete when it returns
inline int finish_call(as_ctx *ctx) {
  if (ctx->own_stream) AS_HIP(ctx, hipStreamSynchronize(ctx->stream));
  return AS_OK;
}

// No C++ exception leaves a C entry (allocation of the host's own bookkeeping is all that can throw).
template <class F>
int guarded(as_ctx *ctx, F &&f) {
  try {
    return f();
  } catch (const std::exception &e) {
    try {
      return fail(ctx, AS_ERR_HIP, e.what());
    } catch (...) {
      return AS_ERR_HIP;
    }
  }
}

// ---- element access ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float bf16_to_f32(unsigned short u) { return __uint_as_float((unsigned int)u << 16); }
template <int DT>
__device__ __forceinline__ float load_as_f32(const void *p, size_t i) {
  if constexpr (DT == AS_F64) return (float)((const double *)p)[i];
  else if constexpr (DT == AS_F32) return ((const float *)p)[i];
  else if constexpr (DT == AS_BF16) return bf16_to_f32(((const unsigned short *)p)[i]);
  else return (float)((const _Float16 *)p)[i];
}
template <int DT>
__device__ __forceinline__ void store_from_f32(void *p, size_t i, float v) {
  if constexpr (DT == AS_F32) ((float *)p)[i] = v;
  else if constexpr (DT == AS_BF16) ((__bf16 *)p)[i] = (__bf16)v;
  else ((_Float16 *)p)[i] = (_Float16)v;
}

// Eight consecutive values of a row of any alignment and length as the matrix holds them (16-bit types: w[0]; f32: w[0], w[1]), columns
// behind the row's d as zeros.  A piece that sticks out of its row is read further left, where it ends with the row, and shifted.
template <int DT>
struct Piece8 {
  u32x4 w[DT == AS_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const char *row, uint32_t column, uint32_t d) {
    if constexpr (DT == AS_F32) {
      const float *p = (const float *)row;
      if (d < 4) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 2][e & 3] = column + e < d ? __float_as_uint(p[column + e]) : 0u;
        return;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t c = column + 4 * h, at = c + 4 <= d ? c : d - 4;
        u32x4 x;
        __builtin_memcpy(&x, p + at, 16);
        if (d & 3) {  // (uniform)
          const uint32_t s = c - at;
          x = s == 1 ? u32x4{x[1], x[2], x[3], 0u} : s == 2 ? u32x4{x[2], x[3], 0u, 0u} : s == 3 ? u32x4{x[3], 0u, 0u, 0u} : x;
        }
        w[h] = c < d ? x : u32x4{0u, 0u, 0u, 0u};
      }
    } else {
      const unsigned short *p = (const unsigned short *)row;
      if (d < 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[0][e] = (column + 2 * e < d ? (uint32_t)p[column + 2 * e] : 0u) | (column + 2 * e + 1 < d ? (uint32_t)p[column + 2 * e + 1] << 16 : 0u);
        return;
      }
      const uint32_t at = column + 8 <= d ? column : d - 8;
      u32x4 x;
      __builtin_memcpy(&x, p + at, 16);
      if (d & 7) {  // (uniform)
        const uint32_t s = column < d ? (column - at) * 16 : 0;
        uint64_t lo = (uint64_t)x[0] | (uint64_t)x[1] << 32, hi = (uint64_t)x[2] | (uint64_t)x[3] << 32;
        if (s >= 64) lo = hi, hi = 0;
        const uint32_t r = s & 63;
        lo = lo >> r | (r ? hi << (64 - r) : 0);
        hi >>= r;
        x = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
      }
      w[0] = column < d ? x : u32x4{0u, 0u, 0u, 0u};
    }
  }
};

}  // namespace asx
