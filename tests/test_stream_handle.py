"""The binding's stream argument: None is torch's current stream of the calling
thread, whatever stream or thread that is. A workspace that the binding allocates
belongs to the call's stream."""

import threading

import pytest
import torch

from flint_amd.flint_lib import Flint, stream_handle

pytestmark = pytest.mark.gpu


def test_none_is_the_current_stream(cuda):
    side = torch.cuda.Stream()
    for _ in range(2):   # the first call initialises, later ones ask torch directly
        assert stream_handle(None) == torch.cuda.current_stream().cuda_stream
        with torch.cuda.stream(side):
            assert stream_handle(None) == side.cuda_stream
            seen = []
            other = threading.Thread(
                target=lambda: seen.append((stream_handle(None),
                                            torch.cuda.current_stream().cuda_stream)))
            other.start()
            other.join()
            assert seen[0][0] == seen[0][1] != side.cuda_stream
        assert stream_handle(None) == torch.cuda.current_stream().cuda_stream
    assert stream_handle(side) == side.cuda_stream
    assert stream_handle(5) == 5


class Noted:
    """The library with some functions noted instead of called."""

    def __init__(self, lib):
        self.lib, self.calls = lib, []

    def __getattr__(self, name):
        if name.endswith(("_workspace", "_last_error", "_string")):
            return getattr(self.lib, name)
        return lambda *args: self.calls.append(args) or 0


A = 0x100000
CALLS = {
    "gemm_tn": lambda f, s: f.gemm_tn(A, A, A, 128, 128, 8192, stream=s),
    "attention_backward": lambda f, s: f.attention_backward(*[A] * 9, 8, 1024, 64, 0.125, stream=s),
    "attention_packed_backward": lambda f, s: f.attention_packed_backward(
        *[A] * 10, f.packed_shape(4096, 3, 8, 2, 64), 0.125, stream=s),
    "attention_paged": lambda f, s: f.attention_paged(
        *[A] * 9, f.paged_shape(4, 4, 1, 8, 2, 64, 512, 128, 512, 999, 64, 200), 0.125, stream=s),
    "bias_gradient": lambda f, s: f.bias_gradient(A, A, 8192, 768, stream=s),
    "layernorm_backward": lambda f, s: f.layernorm_backward(*[A] * 8, 8192, 768, stream=s),
    "embedding_backward": lambda f, s: f.embedding_backward(A, A, A, A, 8, 1024, 50257, 768, stream=s),
}


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_a_workspace_let_go_of_stays_the_streams(cuda, name, handle):
    """Memory of a call on another stream is not given to the current one, whose
    work does not wait for that call."""
    f = Flint()
    f.lib = Noted(f.lib)
    side = torch.cuda.Stream()
    torch.cuda.empty_cache()
    CALLS[name](f, side.cuda_stream if handle else side)
    workspace, size, stream = f.lib.calls[0][-3:]
    assert workspace and size >= 16 and stream == side.cuda_stream
    assert torch.empty(size, dtype=torch.uint8, device=cuda).data_ptr() != workspace
    with torch.cuda.stream(side):   # where it came from, it is free again
        assert torch.empty(size, dtype=torch.uint8, device=cuda).data_ptr() == workspace
