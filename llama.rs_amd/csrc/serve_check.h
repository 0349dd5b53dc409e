// serve_check.h — host-side checks shared by the batched serving operators.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <initializer_list>
#include <string>

#include "../../include/rlh_serve.h"
#include "sampler.h"

namespace rlh {

inline int serve_error(int code, const std::string& msg) { return set_error(code, msg.c_str()); }

inline uint32_t float_type_size(uint32_t ty) {
  return ty == RLH_TYPE_F32 ? 4u : ty == RLH_TYPE_F16 || ty == RLH_TYPE_BF16 ? 2u : 0u;
}

inline bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// Whether [a, a + na) and [b, b + nb) share a byte.
inline bool overlap(const void* a, uint64_t na, const void* b, uint64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + nb && y < x + na;
}

// Bytes from the first to the last value of n rows of `width` values.
inline uint64_t row_bytes_span(uint64_t n, uint64_t stride, uint64_t width, uint32_t size) {
  return n ? ((n - 1) * stride + width) * size : 0;
}

// Rows of `width` values of `size` bytes: pointer and stride as the kernels'
// 16-byte accesses need them.
inline int check_rows(const char* name, const void* p, uint64_t stride, uint64_t width, uint32_t size) {
  if (!p) return serve_error(RLH_EINVAL, std::string(name) + " is null");
  if (!aligned(p, 16)) return serve_error(RLH_EINVAL, std::string(name) + " is not aligned to 16 bytes");
  if (stride < width) return serve_error(RLH_EINVAL, std::string(name) + ": stride below the row's width");
  if (stride > (1ull << 32)) return serve_error(RLH_EINVAL, std::string(name) + ": stride above 2^32");
  if (stride * size % 16) return serve_error(RLH_EINVAL, std::string(name) + ": stride is not a multiple of 16 bytes");
  return RLH_OK;
}

// Bytes of the pool's k, and of its v; whether [p, p + n) meets one of them.
inline uint64_t pool_bytes(const rlh_kv_pages& kv) {
  return kv.n_pages * kv.n_head_kv * kv.page_size * kv.head_dim * 2;
}
inline bool overlaps_pool(const rlh_kv_pages& kv, const void* p, uint64_t n) {
  return overlap(p, n, kv.k, pool_bytes(kv)) || overlap(p, n, kv.v, pool_bytes(kv));
}

// An argument's memory: `rows` of `width` bytes, `stride` bytes apart.
struct Area {
  const char* name;
  const void* p;
  uint64_t rows, stride, width;
  bool empty() const { return !p || rows == 0 || width == 0; }
  uint64_t span() const { return rows ? (rows - 1) * stride + width : 0; }
};
inline Area area(const char* name, const void* p, uint64_t bytes) { return Area{name, p, 1, bytes, bytes}; }

// Whether they share a byte; what lies between one's rows is not its own (of
// two with gaps, the second counts as a whole).
inline bool meet(const Area& a, const Area& b) {
  if (a.empty() || b.empty() || !overlap(a.p, a.span(), b.p, b.span())) return false;
  if (a.rows == 1 && b.rows > 1) return meet(b, a);
  if ((uintptr_t)b.p < (uintptr_t)a.p) return true;
  const uint64_t off = (uintptr_t)b.p - (uintptr_t)a.p, row = off / a.stride;
  return off % a.stride < a.width || (row + 1 < a.rows && (row + 1) * a.stride < off + b.span());
}
inline int check_apart(const Area& written, std::initializer_list<Area> others) {
  for (const Area& o : others)
    if (meet(written, o)) return serve_error(RLH_EINVAL, std::string(written.name) + " overlaps " + o.name);
  return RLH_OK;
}

// The batch's arrays.
inline Area area_q_start(const rlh_seqs& s) { return area("q_start", s.q_start, ((uint64_t)s.n_seq + 1) * 4); }
inline Area area_kv_len(const rlh_seqs& s) { return area("kv_len", s.kv_len, (uint64_t)s.n_seq * 4); }
inline Area area_table(const rlh_seqs& s, uint32_t page_size) {
  return Area{"table", s.table, s.n_seq, (uint64_t)s.table_stride * 4, ((uint64_t)s.max_kv + page_size - 1) / page_size * 4};
}

// The pool and the batch (no device needed).
int check_batch(const rlh_kv_pages* kv, const rlh_seqs* seqs, uint32_t n_head);

// The current device, then pointers against it. A call's small arrays mostly
// lie in one allocation: what is known of it holds for all of them, which spares
// most of the lookups (a call with seven: 3.7 to 3.3 us of the host's time). Of a
// reserved range that is mapped in pieces the runtime names the pointer's piece.
class DeviceCheck {
 public:
  int begin() {
    if (hipGetDevice(&dev_) == hipSuccess) return RLH_OK;
    (void)hipGetLastError();
    return serve_error(RLH_EDEVICE, "no HIP device available (librlh needs an MI355X / gfx950 GPU)");
  }
  int device() const { return dev_; }
  // nullptr passes: a missing argument is found before
  int operator()(const char* name, const void* p) const {
    if (!p) return RLH_OK;
    for (const Range& r : known_)
      if ((uintptr_t)p - r.base < r.size) return RLH_OK;
    hipPointerAttribute_t a{};
    if (hipPointerGetAttributes(&a, p) != hipSuccess) {
      (void)hipGetLastError();
      return serve_error(RLH_EINVAL, std::string(name) + " is not device-accessible memory");
    }
    if (a.devicePointer == nullptr) return serve_error(RLH_EINVAL, std::string(name) + " is not device-accessible memory");
    if (a.type == hipMemoryTypeDevice && a.device != dev_)
      return serve_error(RLH_EINVAL, std::string(name) + " is memory of another device than the current one");
    if (a.type != hipMemoryTypeDevice) return RLH_OK;
    hipDeviceptr_t base;
    size_t size;
    if (hipMemGetAddressRange(&base, &size, (hipDeviceptr_t)p) == hipSuccess)
      known_[next_++ % 4] = Range{(uintptr_t)base, size};
    else
      (void)hipGetLastError();
    return RLH_OK;
  }

 private:
  struct Range {
    uintptr_t base, size;
  };
  int dev_ = -1;
  mutable Range known_[4] = {};  // device memory that has been looked up
  mutable uint32_t next_ = 0;
};

#define RLH_TRY(expr)            \
  do {                           \
    const int rc_ = (expr);      \
    if (rc_ != RLH_OK) return rc_; \
  } while (0)

// Enqueues a kernel; `what` is the entry that does. The launch's own status
// counts: the thread's last error may be one that the caller left.
template <typename T>
struct as_is {
  typedef T type;
};
template <typename... P>
int enqueue(const char* what, void (*kernel)(P...), dim3 grid, uint32_t threads, uint32_t lds, hipStream_t stream,
            typename as_is<P>::type... args) {
  // (a launch of 2^32 threads or more is not refused: it leaves blocks out)
  if ((uint64_t)grid.x * threads >> 32) return serve_error(RLH_EUNSUP, std::string(what) + ": a launch of 2^32 threads");
  void* p[] = {(void*)&args...};
  const hipError_t e = hipLaunchKernel((const void*)kernel, grid, dim3(threads), p, lds, stream);
  if (e == hipSuccess) return RLH_OK;
  (void)hipGetLastError();
  return serve_error(RLH_EDEVICE, std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace rlh
