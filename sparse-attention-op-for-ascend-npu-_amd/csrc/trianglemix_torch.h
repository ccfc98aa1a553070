// What the files of the torch adapter share.
#ifndef TRIANGLEMIX_TORCH_H
#define TRIANGLEMIX_TORCH_H

#include <ATen/ATen.h>

#include <stdint.h>

namespace trianglemix_rocm {

// Workspace of at least `bytes` for a launch on `stream`: the buffer kept for
// this device and stream, or under stream capture one of the capture's own.  Any
// other launch on the stream may use it too: it holds nothing between launches.
at::Tensor workspace_for(const at::Tensor& like, int64_t bytes, void* stream);

// Raises the library's last error unless the status is TM_OK.
void check_status(int status, const char* what);

}  // namespace trianglemix_rocm

#endif  // TRIANGLEMIX_TORCH_H
