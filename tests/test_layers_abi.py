"""The argument blocks of the calls around the head: their layouts as a C compiler sees them, and what
the host refuses without a GPU."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"lily_norm_args_t": "NormArgs", "lily_linear_args_t": "LinearArgs", "lily_adjust_args_t": "AdjustArgs"}


def test_layouts_are_those_of_the_headers(lily, tmp_path):
    lines = []
    for c, py in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in getattr(lily, py)._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "lily_layers.h"\nint main(void) {'
                   + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o",
                    str(tmp_path / "layout"), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in STRUCTS.values():
        t = getattr(lily, py)
        want += [C.sizeof(t)] + [getattr(t, f[0]).offset for f in t._fields_]
    assert got == want


def test_no_handle_is_refused(lily):
    for call, args in (("lily_add_rms_norm", lily.NormArgs()), ("lily_linear", lily.LinearArgs()),
                       ("lily_adjust_logits", lily.AdjustArgs())):
        assert getattr(lily.lib(), call)(None, None, C.byref(args)) == lily.ERR_ARG


def test_tensors_that_are_not_in_order_are_named(lily):
    import torch

    host = torch.zeros((2, 8))
    with pytest.raises(lily.LilyError, match="x must be a tensor on the handle's device"):
        lily._Rows("x", host, 0, (torch.float32,))
    with pytest.raises(lily.LilyError, match="bias"):
        lily._Rows("bias", [1.0], 0, (torch.float32,))
    assert lily._Rows("bias", None, 0, (torch.float32,)).p is None
    assert lily.ACTIVATIONS == {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
