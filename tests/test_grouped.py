"""What the products by runs of rows refuse, before anything touches a device."""

import ctypes
import inspect
import pathlib
import subprocess
import sys

import pytest
import torch

from ninetoothed_b200 import _capi


def h(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


def bounds(*values):
    return torch.tensor(values, dtype=torch.int32)


GROUPED = dict(lhs=h(6, 8), rhs=h(2, 8, 16), offsets=bounds(0, 2, 6), output=h(6, 16))
GRAD = dict(lhs=h(6, 8), output_grad=h(6, 16), offsets=bounds(0, 2, 6), rhs_grad=h(2, 8, 16))
LORA = dict(lhs=h(6, 8), rhs=h(8, 16), down=h(3, 8, 8), up=h(3, 8, 16), scales=torch.ones(3), offsets=bounds(0, 2, 6),
            adapters=bounds(2, -1), output=h(6, 16))
CALLS = [(_capi.grouped_matmul, GROUPED), (_capi.grouped_matmul_rhs_grad, GRAD), (_capi.lora_matmul, LORA)]


@pytest.mark.parametrize("function, good", CALLS)
def test_well_formed_calls_get_as_far_as_the_device_check(function, good):
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        function(**good)


@pytest.mark.parametrize("function, good", CALLS)
def test_every_tensor_is_checked_for_rank_type_and_being_one(function, good):
    for name, tensor in good.items():
        with pytest.raises(TypeError):
            function(**{**good, name: None})
        with pytest.raises(ValueError):
            function(**{**good, name: tensor[None]})
        with pytest.raises(TypeError):
            function(**{**good, name: tensor.double()})
    for name in ("offsets", "adapters"):
        if name in good:
            with pytest.raises(TypeError, match="int32 or torch.int64"):
                function(**{**good, name: good[name].to(torch.int16)})
            with pytest.raises(RuntimeError, match="CUDA tensors only"):
                function(**{**good, name: good[name].long()})


def test_the_slow_path_warning_names_the_call(monkeypatch):
    """Whatever frames of this package and of PyTorch lie between the call and the warning."""
    class Library:
        launches = 10 ** 9

        def ninetoothed_b200_plain_launches(self, reset):
            self.launches += 1
            return self.launches

        def ninetoothed_b200_last_note(self):
            return b"slow"

    fake = Library()
    monkeypatch.setattr(_capi, "library", lambda: fake)
    monkeypatch.setattr(_capi, "_plain_launches_seen", 0)
    names = {"warn": _capi.warn_of_plain_launches}
    inner, outer = pathlib.Path(_capi.__file__).with_name("torch_ops.py"), pathlib.Path(torch.__file__).with_name("_ops.py")
    exec(compile("def through_package(): warn()", str(inner), "exec"), names)
    exec(compile("def through_torch(): through_package()", str(outer), "exec"), names)
    for call in (names["warn"], names["through_package"], names["through_torch"]):
        with pytest.warns(_capi.SlowPathWarning, match="slow") as caught:
            call()
        assert caught[0].filename == __file__
        assert caught[0].lineno == inspect.currentframe().f_lineno - 2


def test_the_operators_library_is_tied_to_its_pytorch(monkeypatch, tmp_path):
    assert _capi.torch_library_fits()  # as built
    monkeypatch.setattr(_capi, "TORCH_LIBRARY_PATH", tmp_path / "lib.so")
    assert not _capi.torch_library_fits()
    _capi.TORCH_LIBRARY_PATH.write_bytes(b"no library")
    assert not _capi.torch_library_fits()  # nothing says what it was built with
    _capi.torch_version_record().write_text("0.1\n")
    assert not _capi.torch_library_fits()
    _capi.torch_version_record().write_text(f"{torch.__version__}\n")
    assert _capi.torch_library_fits()


def test_the_operators_import_beside_a_library_of_another_pytorch(tmp_path):
    (tmp_path / "lib.so").write_bytes(b"no library")
    (tmp_path / "lib.torch-version").write_text("0.1\n")
    program = (f"import pathlib, torch; from ninetoothed_b200 import _capi\n"
               f"_capi.TORCH_LIBRARY_PATH = pathlib.Path({str(tmp_path / 'lib.so')!r})\n"
               "import ninetoothed_b200.torch_ops\n"
               "for name in ('matmul', 'softmax', 'grouped_matmul', 'grouped_matmul_rhs_grad', 'lora_matmul'):\n"
               "    assert torch._C._dispatch_has_kernel_for_dispatch_key(f'ninetoothed_b200::{name}', 'CUDA'), name\n")
    subprocess.run([sys.executable, "-c", program], check=True, cwd=pathlib.Path(_capi.__file__).resolve().parent.parent)


def launch(name, tensors, *trailing):
    kept = [_capi.tensor_arg(t) for t in tensors]
    return getattr(_capi.library(), name)(None, *(k[0] for k in kept), *trailing)


def launch_lora(workspace_size=1 << 20, workspace=256, dtypes=(8, 2, 2), **changed):
    return launch("launch_lora_matmul", {**LORA, **changed}.values(), *dtypes, ctypes.c_void_p(workspace),
                  ctypes.c_size_t(workspace_size))


def test_the_entry_points_refuse_shapes_that_do_not_agree():
    for name, good, changes in (
            ("launch_grouped_matmul", GROUPED, [dict(lhs=h(6, 16)), dict(output=h(5, 16)), dict(output=h(6, 8)),
                                                dict(offsets=bounds(0, 6)), dict(rhs=h(2, 7, 16))]),
            ("launch_grouped_matmul_rhs_grad", GRAD, [dict(lhs=h(5, 8)), dict(rhs_grad=h(2, 16, 8)),
                                                      dict(rhs_grad=h(3, 8, 16)), dict(offsets=bounds(0, 1, 2, 6))])):
        for change in changes:
            assert launch(name, {**good, **change}.values(), 8, 2) == -2, (name, change)
    for change in (dict(rhs=h(7, 16)), dict(down=h(3, 7, 8)), dict(up=h(2, 8, 16)), dict(up=h(3, 7, 16)),
                   dict(up=h(3, 8, 15)), dict(scales=torch.ones(2)), dict(offsets=bounds(0, 6)),
                   dict(adapters=bounds(0, 1, 2)), dict(output=h(6, 15)), dict(output=h(7, 16))):
        assert launch_lora(**change) == -2, change


def test_the_entry_points_refuse_types_and_counts_they_do_not_hold():
    assert launch("launch_grouped_matmul", GROUPED.values(), 10, 2) == -1     # float32 operands
    assert launch("launch_grouped_matmul", GROUPED.values(), 8, 1) == -1      # int16 bounds
    assert launch("launch_grouped_matmul_rhs_grad", GRAD.values(), 100, 2) == -1
    assert launch_lora(dtypes=(8, 2, 0)) == -1                                # int8 adapters
    many = 2049
    assert launch("launch_grouped_matmul", [h(6, 8), h(many, 8, 16), torch.zeros(many + 1, dtype=torch.int32), h(6, 16)],
                  8, 2) == -2
    assert b"2048" in _capi.library().ninetoothed_b200_last_error()


def test_the_adapters_workspace():
    size = _capi.lora_matmul_workspace_size(LORA["lhs"], LORA["down"])
    assert size == 6 * 32 * 4
    assert _capi.lora_matmul_workspace_size(h(6, 8), h(3, 8, 33)) == 2 * size
    assert launch_lora(workspace_size=size - 1) == -4
    assert launch_lora(workspace=0) == -4
    assert launch_lora(workspace=264) == -4     # not 256-byte aligned
    with pytest.raises(ValueError, match="must have 3 dimensions"):
        _capi.lora_matmul_workspace_size(h(6, 8), h(8, 8))


def test_the_workspace_tells_which_way_the_adapters_go():
    """A row at a time takes partial sums of its own, one for every 2048 terms; by tiles takes 32 ranks of 32 bits a row."""
    def size(rows, rank):
        return _capi.lora_matmul_workspace_size(h(1, 1).expand(rows, 20480), h(1, 1, 1).expand(2, 20480, rank))

    assert size(6000, 16) == 10 * 6000 * 16 * 4     # 2048 requests of three rows: 1394 us a row at a time, 1669 by tiles
    assert size(8192, 16) == 8192 * 32 * 4          # of four rows: 1895 and 1661


def test_nothing_to_do_needs_no_device():
    assert launch("launch_grouped_matmul", [h(0, 8), h(2, 8, 16), bounds(0, 0, 0), h(0, 16)], 8, 2) == 0
    assert launch("launch_grouped_matmul", [h(6, 8), h(0, 8, 16), bounds(0), h(6, 16)], 8, 2) == 0
    assert launch("launch_grouped_matmul_rhs_grad", [h(6, 0), h(6, 16), bounds(0, 2, 6), h(2, 0, 16)], 8, 2) == 0
    assert launch_lora(lhs=h(0, 8), output=h(0, 16)) == 0
    assert launch_lora(adapters=bounds(), offsets=bounds(0)) == 0
