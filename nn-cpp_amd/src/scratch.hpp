// scratch.hpp - a call's device scratch, also while its stream is captured into a graph (internal to libnnh).
//
// Outside a capture it is the stream's StreamWorkspace, its size checked first. A captured launch keeps the address it was
// given for as long as the graph lives, so the library's own buffer, which may grow and move, is no place for it, and an
// event recorded in a capture cannot order later eager work: a captured call takes the buffer that the caller registered
// for the stream (nnh_set_workspace) and is refused without one. Graphs that may run at once need a buffer each.
//
// The kernels move scratch in words of up to 16 bytes, into LDS and through scalar registers too, which take no other address: a
// registered buffer that begins elsewhere is refused.
#pragma once

#include <hip/hip_runtime.h>

#include <optional>

#include "abi_common.hpp"
#include "workspace.hpp"

namespace nnh {

class Scratch {
public:
	Scratch(hipStream_t s, size_t bytes) {
		if (bytes == 0) return;
		hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
		status_ = hip_status(hipStreamIsCapturing(s, &capture), "capture status");
		if (status_ != NNH_OK) return;
		if (capture != hipStreamCaptureStatusNone) {
			size_t have = 0;
			status_ = hip_status(registered_workspace(s, base_, have), "workspace lookup");
			if (status_ == NNH_OK && (!base_ || have < bytes))
				status_ = fail(NNH_ERR_WORKSPACE, "a call captured into a graph needs a registered workspace of " + std::to_string(bytes) + " bytes");
			check_place();
			return;
		}
		status_ = check_workspace(s, bytes);
		if (status_ != NNH_OK) return;
		own_.emplace(s, bytes);
		status_ = hip_status(own_->error(), "workspace");
		if (status_ == NNH_OK) base_ = own_->at<void>(0);
		check_place();
	}
	int status() const { return status_; }
	template <typename T>
	T* at(size_t offset) const {
		return base_ ? reinterpret_cast<T*>(static_cast<char*>(base_) + offset) : nullptr;
	}

private:
	void check_place() {
		if (status_ == NNH_OK && reinterpret_cast<uintptr_t>(base_) % 16 != 0)
			status_ = fail(NNH_ERR_WORKSPACE, "the registered workspace must begin at a multiple of 16 bytes");
	}

	int status_ = NNH_OK;
	void* base_ = nullptr;
	std::optional<StreamWorkspace> own_;
};

}  // namespace nnh
