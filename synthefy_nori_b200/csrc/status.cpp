// The status word of a device, made while a CUDA graph is being captured.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

namespace nori {

// One int32, zeroed now and in memory of its own: on the capturing stream its memory would be the graph's, and every
// replay would clear it, whatever a kernel has reported.
torch::Tensor status_word_beside_capture(int64_t device) {
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
  const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
  for (int i = 0; i < 64; ++i) {  // (streams of the pool in turn: the capturing one may be among them)
    const auto side = at::cuda::getStreamFromPool(false, static_cast<c10::DeviceIndex>(device));
    cudaStreamCaptureStatus capturing;
    C10_CUDA_CHECK(cudaStreamIsCapturing(side.stream(), &capturing));
    if (capturing != cudaStreamCaptureStatusNone) continue;
    const c10::cuda::CUDAStreamGuard on(side);
    auto word = torch::zeros({1}, torch::dtype(torch::kInt32).device(torch::kCUDA, static_cast<c10::DeviceIndex>(device)));
    C10_CUDA_CHECK(cudaStreamSynchronize(side.stream()));
    return word;
  }
  TORCH_CHECK(false, "status word: every stream of the pool is being captured");
}

}  // namespace nori
