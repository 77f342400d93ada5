"""The language-model operators without a GPU: the C entry points' checks and plans (operators_host.cpp, under
AddressSanitizer and UndefinedBehaviorSanitizer), and what the Python side refuses before it calls them."""

import os
import re
import subprocess

import pytest

from harp_amd import build, operators as ops
from harp_amd.backend import HipBuffer
from harp_amd.frontend import DType, F32, I32


def test_entry_points_and_plans():
    r = subprocess.run([build.build_operator_checks()], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    assert r.stdout.strip().endswith(" 0 failed")


@pytest.mark.parametrize("source", ["gated_scan", "token_rows"])
def test_no_shift_by_the_last_register(source, tmp_path):
    """A 64-bit shift whose amount is in the last register of a kernel's allocation was seen to take another
    register's value for it: no kernel has one."""
    out = str(tmp_path / "code.s")
    subprocess.run([os.path.join(build.ROCM, "bin", "hipcc"), "-std=c++17", *build.DEVICE_FLAGS, "--offload-device-only", "-S",
                    os.path.join(build.CSRC, "kernels", source + ".hip"), "-o", out], check=True, capture_output=True, timeout=300)
    with open(out) as f:
        kernels = re.findall(r"\n(_Z\S+):(.*?)\.amdhsa_next_free_vgpr (\d+)", f.read(), re.S)
    assert kernels
    for name, code, registers in kernels:
        last = (int(registers) + 7) // 8 * 8 - 1
        assert not re.search(r"v_(lshlrev|lshrrev|ashrrev)_[bi]64\S* v\[\d+:\d+\], v%d," % last, code), name


class Tensor:
    """What the operators look at of another library's tensor."""

    def __init__(self, shape, dtype="torch.float32", strides=None, gpu=0, address=4096):
        self.shape, self.dtype = tuple(shape), dtype
        self._strides, self._gpu, self._address = strides or ops._dense(self.shape), gpu, address

    def data_ptr(self):
        return self._address

    def stride(self):
        return self._strides

    def get_device(self):
        return self._gpu


class Device:
    index = 0


class Handle:
    value = 77


class Buffer(HipBuffer):
    def __init__(self, device, shape, dtype):
        self.device, self.shape, self.dtype, self._h = device, list(shape), dtype, Handle()

    def __del__(self):
        pass


def buffer(device, shape, dtype=F32):
    return Buffer(device, shape, dtype)


def test_fields_of_an_array():
    d = Device()
    assert ops._array(d, Tensor([3, 5]), "a", 2) == ((3, 5), 0, (0, 4096, 60, 5, 0, 0))
    assert ops._array(d, Tensor([3, 5], "torch.bfloat16", (9, 1)), "a", 2)[2] == (0, 4096, 2 * (2 * 9 + 5), 9, 0, 1)
    assert ops._array(d, Tensor([2, 3, 4], "torch.float16", (0, 8, 1)), "a", 3)[2] == (0, 4096, 2 * (2 * 8 + 4), 0, 8, 2)
    assert ops._array(d, Tensor([0, 5], address=0), "a", 2)[2][1] != 0           # an empty array is not an absent one
    assert ops._array(d, Tensor([3, 1], strides=(7, 99)), "a", 2)[2][3] == 7     # one column: its stride does not matter
    b = buffer(d, [2, 3])
    assert ops._array(d, b, "a", 2)[2] == (77, 0, 0, 3, 0, 0)
    assert ops._array(d, ops.View(b, [2, 2], I32, offset=8, strides=[3, 1]), "a", 2)[2] == (77, 8, 0, 3, 0, 3)


@pytest.mark.parametrize("word,make", [
    ("expected 2 axes", lambda d: ops._array(d, Tensor([3]), "a", 2)),
    (r"expected \(4, 5\)", lambda d: ops._array(d, Tensor([3, 5]), "a", 2, (4, 5))),
    ("last axis", lambda d: ops._array(d, Tensor([3, 5], strides=(1, 3)), "a", 2)),
    ("last axis", lambda d: ops._array(d, Tensor([3, 5, 2], strides=(10, 1, 5)), "a", 3)),
    ("contiguous", lambda d: ops._array(d, Tensor([3], strides=(2,)), "a", 1)),
    ("not supported", lambda d: ops._array(d, Tensor([3], "torch.float64"), "a", 1)),
    ("the host", lambda d: ops._array(d, Tensor([3], gpu=-1), "a", 1)),
    ("GPU 1", lambda d: ops._array(d, Tensor([3], gpu=1), "a", 1)),
    ("no array", lambda d: ops._array(d, [1.0, 2.0], "a", 1)),
    ("another device handle", lambda d: ops._array(d, buffer(Device(), [3]), "a", 1)),
    ("no element type", lambda d: ops._array(d, buffer(d, [3], None), "a", 1)),
    ("not supported", lambda d: ops._array(d, buffer(d, [3], DType("f64")), "a", 1)),
    ("before its buffer", lambda d: ops._array(d, ops.View(buffer(d, [3]), [3], F32, offset=-4), "a", 1)),
    ("as many strides", lambda d: ops.View(buffer(d, [3]), [3], F32, strides=[1, 1])),
    ("has to be f32", lambda d: ops._small(d, Tensor([3], "torch.float16"), "a", (3,), 0)),
    ("has to be contiguous", lambda d: ops._small(d, Tensor([3, 2], strides=(4, 1)), "a", (3, 2), 0)),
    ("entropy", lambda d: ops.token_logprobs_backward(d, Tensor([3, 5]), Tensor([3], "torch.int64"), Tensor([3, 2]), grad_entropy=Tensor([3]), out=Tensor([3, 5]))),
    ("rows", lambda d: ops.distill_loss(d, Tensor([3, 5]), Tensor([4, 2]), Tensor([4, 2], "torch.int32"), out=ops.Distilled(Tensor([3]), Tensor([3, 2]), None))),
    ("top_logp", lambda d: ops.token_logprobs(d, Tensor([3, 5]), Tensor([3], "torch.int64"), top=2, out=ops.Logprobs(Tensor([3]), None, Tensor([3, 2]), None, None))),
    ("grad", lambda d: ops.distill_loss(d, Tensor([3, 5]), Tensor([3, 2]), Tensor([3, 2], "torch.int32"), grad=True, out=ops.Distilled(Tensor([3]), Tensor([3, 2]), None))),
])
def test_refused_before_the_call(word, make):
    with pytest.raises((ValueError, TypeError), match=word):
        make(Device())
