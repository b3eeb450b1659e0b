/* What the entry points of include/d3s_train.h and include/d3s_step.h share: the
 * workspace's two sources, the stream's lock, small checks.  Host code only. */
#ifndef D3S_ROOM_H
#define D3S_ROOM_H

#include "d3s_train_internal.h"

namespace d3s {
namespace {

int done() { return hipGetLastError() == hipSuccess ? D3S_OK : D3S_ERR_LAUNCH; }

/* f() under the stream's lock; host memory that runs out (the lock's table) is a status, not an exception */
template <class F>
int locked(void *stream, F f) {
  try {
    const auto lock = d3s::stream_call_lock((hipStream_t)stream);
    return f();
  } catch (...) {
    return D3S_ERR_NOMEM;
  }
}

constexpr int64_t INT_MOST = 0x7fffffff;

/* Where a call's workspace comes from: the caller, or the stream's block. */
struct Room {
  bool given;
  void *ptr;
  int64_t bytes;
};

/* *out: `need` bytes (null for 0); a status when they are not to be had */
int take_room(const Room &r, size_t need, hipStream_t s, void **out) {
  *out = nullptr;
  if (r.given && r.bytes < 0) return D3S_ERR_ARG;
  if (need == 0) return D3S_OK;
  if (!r.given) {
    /* a graph may be replayed beside other calls on the stream, or outlive its
     * block: capture takes a workspace of the caller's */
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &st) != hipSuccess) {
      (void)hipGetLastError();
      return D3S_ERR_LAUNCH;
    }
    if (st != hipStreamCaptureStatusNone) return D3S_ERR_WORKSPACE;
    *out = d3s::stream_workspace(s, need);
    if (!*out) (void)hipGetLastError();
    return *out ? D3S_OK : D3S_ERR_NOMEM;
  }
  if (!r.ptr || (size_t)r.bytes < need) return D3S_ERR_WORKSPACE;
  if ((uintptr_t)r.ptr % 256u != 0u) return D3S_ERR_ARG;
  *out = r.ptr;
  return D3S_OK;
}

size_t size_of(int dtype) { return dtype == D3S_DTYPE_F32 ? 4u : 2u; }
bool known(int dtype) { return dtype == D3S_DTYPE_F32 || dtype == D3S_DTYPE_BF16; }
bool off(const void *p, size_t size) { return (uintptr_t)p % size != 0u; }
Dtype type_of(int dtype) { return dtype == D3S_DTYPE_F32 ? DT_F32 : DT_BF16; }

}  // namespace
}  // namespace d3s

#endif
