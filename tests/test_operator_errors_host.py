"""Which errors of the compiled operators become the package's own exception: what the library refused, nothing else."""

import pytest
import torch


def raising(error):
    def op(*args):
        raise error

    return op


class DriverError(RuntimeError):
    """Stands for a CUDA error, which PyTorch raises as a type of its own."""


@pytest.mark.parametrize("error", [torch.OutOfMemoryError("CUDA out of memory.\nTried to allocate"), DriverError("CUDA error\nmore"),
                                   NotImplementedError("x"), ValueError("y"), RuntimeError("Inference tensors cannot be saved\nfor backward")])
def test_other_errors_keep_their_kind_and_text(monkeypatch, error):
    import coda_kernels_b200 as ck
    from coda_kernels_b200 import ops_rows

    monkeypatch.setitem(ops_rows._native_ops, "rms_norm", raising(error))
    with pytest.raises(type(error)) as caught:
        ops_rows.call_native("rms_norm")
    assert caught.value is error and not isinstance(caught.value, ck.CodaB200Error)


def test_what_the_library_refuses_is_the_packages_error(monkeypatch):
    import coda_kernels_b200 as ck
    from coda_kernels_b200 import ops_rows

    monkeypatch.setitem(ops_rows._native_ops, "rms_norm", raising(RuntimeError("add_rmsnorm failed (code -1): NULL pointer\nC++ frames")))
    with pytest.raises(ck.CodaB200Error, match=r"^add_rmsnorm failed \(code -1\): NULL pointer$"):
        ops_rows.call_native("rms_norm")


@pytest.mark.parametrize("error", [torch.OutOfMemoryError("CUDA out of memory.\nTried to allocate"), DriverError("CUDA error\nmore")])
def test_the_other_compiled_operators_too(monkeypatch, error):
    from coda_kernels_b200 import ops

    if ops._native is None:
        pytest.skip("ctypes dispatch has no compiled operators")
    name = f"stub_that_raises_{type(error).__name__}"  # (the wrapper keeps what it has looked up)
    monkeypatch.setattr(torch.ops.coda_b200n, name, raising(error), raising=False)
    with pytest.raises(type(error)) as caught:
        getattr(ops._native, name)()
    assert caught.value is error
