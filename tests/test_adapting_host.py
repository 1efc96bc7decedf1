"""Adapters, loss and clipping: what needs no GPU.  Structures against the header, argument checks, sizes, refusals."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD_ARG, UNSUPPORTED, ALIGN, RANGE, SCRATCH = "bad argument", "unsupported", "align", "range", "scratch"


def _fields(name):
    """Names of a structure's fields in the header, in their order."""
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "deepshift_b200.h")).read(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} %s;" % name, text).group(1)
    return [f.strip().split()[-1].lstrip("*") for line in body.split(";") if line.strip() for f in line.split(",")]


@pytest.mark.parametrize("name", ["Adapters", "Loss"])
def test_structures_are_those_of_the_header(name, tmp_path):
    from deepshift_b200 import _ffi
    kind = getattr(_ffi, name)
    c_name = "ds_%s_t" % name.lower()
    names = _fields(c_name)
    assert names == [f for f, _ in kind._fields_]
    source = tmp_path / "s.c"
    source.write_text('#include <stdio.h>\n#include <stddef.h>\n#include <stdint.h>\n#include "deepshift_b200.h"\nint main(void) { printf("%%d", (int)sizeof(%s)); %s return 0; }\n'
                      % (c_name, "".join('printf(" %%d", (int)offsetof(%s, %s)); ' % (c_name, f) for f in names)))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "s"), str(source)], check=True)
    size, *offsets = map(int, subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split())
    assert size == ctypes.sizeof(kind) and offsets == [getattr(kind, f).offset for f in names]
    # packed by position, as the calls are
    pack = getattr(_ffi, "pack_" + name.lower())
    values = list(range(1, len(names) + 1))
    got = kind.from_buffer_copy(pack(*values))
    assert [getattr(got, f) for f in names] == values


def _status(text):
    from deepshift_b200 import _ffi
    return [s for s in range(1, 12) if text in _ffi.lib().ds_strerror(s).decode().lower()]


def test_entry_points_check_their_arguments_first():
    from deepshift_b200 import _ffi
    lib = _ffi.lib()
    assert lib.ds_rows_plan(None, 4, 2, None, 0, None) in _status(BAD_ARG)
    assert lib.ds_rows_plan(16, 4, 0, 16, 1 << 20, None) in _status(BAD_ARG)
    assert lib.ds_rows_plan(16, 4, 2, 16, 8, None) not in (0,)   # a plan of eight bytes is too small
    fields = [f for f, _ in _ffi.Adapters._fields_]
    good = dict.fromkeys(fields, 0)
    good.update(rows=4, k=8, n=8, rank=4, count=2, plan=16, down=16, up=16, x=16, x_stride=8, out=16, out_stride=8, h=16, h_bytes=4 * 8 * 4)
    for bad in (dict(rows=-1), dict(k=0), dict(n=0), dict(rank=0), dict(count=0), dict(plan=0), dict(down=0), dict(up=0), dict(x=0), dict(h=0, rank=65, h_bytes=1 << 20), dict(out=0),
                dict(rank=257), dict(count=65536), dict(rows=(1 << 24) + 1), dict(k=(1 << 20) + 1), dict(n=(1 << 20) + 1)):
        assert lib.ds_adapters_apply(_ffi.pack_adapters(*{**good, **bad}.values()), None) != 0, bad
        assert lib.ds_adapters_backward(_ffi.pack_adapters(*{**good, **bad}.values()), None) != 0, bad
    assert lib.ds_adapters_apply(None, None) in _status(BAD_ARG)
    fields = [f for f, _ in _ffi.Loss._fields_]
    good = dict.fromkeys(fields, 0)
    good.update(rows=4, d=8, v=10, type=_ffi.T_BF16, hidden=16, weight=16, target=16, each=16, lse=16, loss=16, count=16, reduction=1, scratch=256, scratch_bytes=1 << 30)
    for bad in (dict(rows=-1), dict(d=0), dict(v=0), dict(type=_ffi.T_F32), dict(type=7), dict(reduction=3), dict(reduction=-1), dict(weight=0), dict(hidden=0), dict(target=0),
                dict(lse=0), dict(count=0), dict(each=0, grad=0), dict(rows=(1 << 24) + 1), dict(v=(1 << 24) + 1), dict(d=(1 << 20) + 1)):
        assert lib.ds_loss_forward(_ffi.pack_loss(*{**good, **bad}.values()), None) != 0, bad
        assert lib.ds_loss_backward(_ffi.pack_loss(*{**good, **bad}.values()), None) != 0, bad
    assert lib.ds_loss_forward(None, None) in _status(BAD_ARG)
    assert lib.ds_clip_norm(None, 1, 1.0, 16, 16, 1 << 20, None) in _status(BAD_ARG)
    table = (ctypes.c_longlong * 4)(16, 16, 4, 0)
    for args in ((-1, 1.0, 16, 16, 1 << 20), (1, -1.0, 16, 16, 1 << 20), (1, math.nan, 16, 16, 1 << 20), (1, 1.0, None, 16, 1 << 20), (1, 1.0, 16, None, 1 << 20), (1, 1.0, 16, 16, 0)):
        assert lib.ds_clip_norm(table, *args, None) != 0, args


def test_sizes():
    from deepshift_b200 import _ffi
    lib = _ffi.lib()
    # a plan: four words, the adapters' first positions, tiles of four words, the rows; behind it the sorting's scratch: rows and counts again
    for rows, count in ((0, 1), (1, 1), (16, 3), (512, 65535), (513, 2), (4096, 64), (1 << 24, 65535)):
        tile = 16 if rows <= 512 else 128
        least = 4 * (4 + count + 2 + 4 * -(-rows // tile) + rows)
        assert least <= lib.ds_rows_plan_bytes(rows, count) <= least + 4 * (4 * min(rows, count + 1) + 8 + rows + count + 2), (rows, count)
    assert lib.ds_adapters_h_bytes(10, 5) == 4 * 10 * 8 and lib.ds_adapters_h_bytes(10, 16) == 4 * 10 * 16
    # the loss keeps no logits (eight bytes for 64 of them at most, and a few for each row), and of their gradients 256 MB at most (or 2048 columns)
    rows, v = 8192, 131072
    assert lib.ds_loss_bytes(rows, 4096, v, 0, 0) <= rows * v // 8 + 16 * rows
    assert lib.ds_loss_bytes(rows, 4096, v, 1, 0) < (256 << 20) + 4 * rows * 4096 + (1 << 20)
    assert lib.ds_loss_bytes(rows, 4096, v, 0, 1) - lib.ds_loss_bytes(rows, 4096, v, 0, 0) >= 2 * 4096 * (rows + v)


def test_refusals_without_a_gpu():
    from deepshift_b200 import adapters, gradients, losses
    for ids, count in (([0, 1], 0), ([0, 2], 2), ([-2], 2), (torch.zeros(2, 2, dtype=torch.int64), 2), (torch.zeros(3), 2), ([0], 65536)):
        with pytest.raises(RuntimeError):
            adapters.plan_rows(ids, count)
    with pytest.raises(RuntimeError, match="CUDA"):
        adapters.apply(torch.zeros(2, 8), torch.zeros(1, 4, 8), torch.zeros(1, 4, 8), None, None)
    h, w, t = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(10, 8, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        losses.linear_cross_entropy(h, w, t)
    with pytest.raises(ValueError, match="reduction"):
        losses.linear_cross_entropy(h, w, t, reduction="average")
    with pytest.raises(RuntimeError, match="CUDA"):
        gradients.clip_norm([torch.zeros(3)], 1.0)
    for worst in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            gradients.clip_norm([], worst)
    with pytest.raises(RuntimeError, match="places"):
        gradients.clip_norm([torch.zeros(3)], 1.0, out=[])
    assert float(gradients.clip_norm([], 1.0)) == 0 and float(gradients.clip_grad_norm_(torch.nn.Parameter(torch.zeros(2)), 1.0)) == 0


def test_an_adapted_layer_starts_as_its_base():
    from deepshift_b200 import adapters
    base = torch.nn.Linear(6, 5)
    layer = adapters.AdaptedLinear(base, count=3, rank=2, alpha=4)
    assert layer.down.shape == (3, 2, 6) and layer.up.shape == (3, 2, 5) and not layer.up.any()
    assert layer.scale.tolist() == [2.0] * 3
    assert [n for n, p in layer.named_parameters() if p.requires_grad] == ["down", "up"]
    assert "count=3, rank=2" in repr(layer)
