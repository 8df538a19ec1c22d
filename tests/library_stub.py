"""The Python side of the operators without a GPU: CPU tensors go through the entry
points, and calls into the library are recorded instead of made."""
import contextlib

import torch

from memoryefficientclip_amd import _function, _lib, _vocab


class Library:
    """Records calls: ``calls[name]`` is the list of their arguments.  No call wants scratch, and the
    contrastive losses' plan is a workspace of one number."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        if not name.startswith("mec_"):
            raise AttributeError(name)

        def call(*args):
            self.calls.setdefault(name, []).append(args)
            return 1 << 4 if name == "mec_forward_plan" else 0

        return call


def install(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_vocab, "check_gpu", lambda *a: None)
    monkeypatch.setattr(_vocab, "launch", lambda index, nbytes, call: call(0, 0))
    monkeypatch.setattr(_function, "check_inputs", lambda x, y: None)
    monkeypatch.setattr(_function, "_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    return lib


@contextlib.contextmanager
def copying_hooks(unpack=lambda t: t):
    """Saved tensors come back as dense copies (what torch.autograd.graph.save_on_cpu makes of
    them), changed by `unpack`; yields the list of those."""
    back = []

    def copy(t):
        back.append(unpack(torch.empty(t.shape, dtype=t.dtype).copy_(t)))
        return back[-1]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), copy):
        yield back


def rows_at(tensors, pointer, rows, inner, outer_stride, inner_stride, size):
    """The rows that a kernel reads from `pointer`, which has to lie in one of `tensors` with all of them."""
    for t in tensors:
        begin = t.untyped_storage().data_ptr()
        end = begin + t.untyped_storage().nbytes()
        if not begin <= pointer < end:
            continue
        last = (rows - 1) // inner * outer_stride + (rows - 1) % inner * inner_stride + size
        assert pointer + last * t.element_size() <= end, "rows beyond the tensor's memory"
        flat = t.as_strided(((end - begin) // t.element_size(),), (1,), 0)
        at = (pointer - begin) // t.element_size()
        return torch.stack([flat[at + q:at + q + size] for q in (r // inner * outer_stride + r % inner * inner_stride
                                                                 for r in range(rows))])
    raise AssertionError("the pointer lies in none of the tensors")
