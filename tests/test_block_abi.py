"""CPU: the block operators' C ABI (include/helix/helix_block.h) as ctypes and
a C compiler see it, and what of it needs no device."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

from helix_b200 import abi

ROOT = Path(__file__).resolve().parent.parent
STRUCTS = {"helix_rms_norm_desc": abi.RmsNormDesc, "helix_quant8_desc": abi.Quant8Desc,
           "helix_matmul8_desc": abi.Matmul8Desc, "helix_gated_scan_desc": abi.GatedScanDesc}


def test_layouts_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "helix/helix_block.h"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f}));' for f, _ in cls._fields_]
        lines.append('printf("\\n");')
    lines.append('printf("consts %d %d %d %d\\n", HELIX_GROUP, HELIX_GATED_CHUNK, HELIX_SCALE_BLOCKS, HELIX_E4M3);')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run([cc, "-std=c11", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "l")],
                   check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.splitlines()
    for line, (name, cls) in zip(out, STRUCTS.items()):
        want = [name, C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
        assert line.split() == [str(x) for x in want]
    assert out[-1].split()[1:] == [str(x) for x in (abi.HELIX_GROUP, abi.HELIX_GATED_CHUNK, abi.HELIX_SCALE_BLOCKS,
                                                    abi.HELIX_E4M3)]


def test_descriptor_defaults():
    lib = abi.load()
    d = abi.RmsNormDesc()
    lib.helix_rms_norm_desc_init(C.byref(d), 10, 300)
    assert (d.n_row, d.n_col, d.ld_x, d.ld_out, d.ld_scale) == (10, 300, 300, 300, 3)
    assert abs(d.eps - 1e-6) < 1e-12 and d.x_dtype == abi.HELIX_F32
    q = abi.Quant8Desc()
    lib.helix_quant8_desc_init(C.byref(q), 10, 300, abi.HELIX_SCALE_ROWS, True)
    assert (q.ld_x, q.ld_q, q.ld_scale) == (300, 16, 1)
    lib.helix_quant8_desc_init(C.byref(q), 10, 300, abi.HELIX_SCALE_BLOCKS, False)
    assert (q.ld_q, q.ld_scale) == (304, 3)
    m = abi.Matmul8Desc()
    lib.helix_matmul8_desc_init(C.byref(m), 3, 5, 300, abi.HELIX_SCALE_BLOCKS)
    assert (m.ld_a, m.ld_b, m.ld_out, m.ld_a_scale, m.out_dtype) == (304, 304, 5, 3, abi.HELIX_BF16)
    g = abi.GatedScanDesc()
    lib.helix_gated_scan_desc_init(C.byref(g), 7, 3, 20)
    assert (g.s_v, g.seq_dg, g.seq_h1) == (20, 140, 20)


def test_null_arguments():
    lib = abi.load()
    n = abi.NULL_TENSOR
    for init, args in ((lib.helix_rms_norm_desc_init, (1, 1)), (lib.helix_quant8_desc_init, (1, 1, 0, False)),
                       (lib.helix_matmul8_desc_init, (1, 1, 1, 0)), (lib.helix_gated_scan_desc_init, (1, 1, 1))):
        init(None, *args)
    bad = abi.HELIX_ERR_INVALID_ARG
    d, q, m, g = abi.RmsNormDesc(), abi.Quant8Desc(), abi.Matmul8Desc(), abi.GatedScanDesc()
    assert lib.helix_rms_norm_encode(None, None, C.byref(d), *[n] * 7) == bad
    assert lib.helix_rms_norm_grad_encode(None, None, C.byref(d), *[n] * 9) == bad
    assert lib.helix_quant8_encode(None, None, C.byref(q), n, n, n) == bad
    assert lib.helix_matmul8_encode(None, None, C.byref(m), *[n] * 5) == bad
    assert lib.helix_gated_scan_encode(None, None, C.byref(g), *[n] * 7) == bad
    assert lib.helix_gated_scan_grad_encode(None, None, C.byref(g), *[n] * 9) == bad
    assert lib.helix_rms_norm_grad_scratch_size(None, None) == 0
    assert lib.helix_gated_scan_states_size(None) == 0


def test_sizes():
    """States: one f32 per chunk of 128 tokens and channel.  The norm's
    gradient: one partial row of dweight per resident row slot of a 148-SM
    part, never more slots than rows."""
    lib = abi.load()
    g = abi.GatedScanDesc()
    for toks, chunks in ((0, 0), (1, 1), (128, 1), (129, 2), (8192, 64)):
        lib.helix_gated_scan_desc_init(C.byref(g), toks, 3, 20)
        assert lib.helix_gated_scan_states_size(C.byref(g)) == 3 * chunks * 20 * 4
    d = abi.RmsNormDesc()
    lib.helix_rms_norm_desc_init(C.byref(d), 1, 4096)
    assert lib.helix_rms_norm_grad_scratch_size(None, C.byref(d)) == 4096 * 4
    lib.helix_rms_norm_desc_init(C.byref(d), 1 << 20, 4096)
    assert lib.helix_rms_norm_grad_scratch_size(None, C.byref(d)) == 2 * 148 * 4096 * 4
    lib.helix_rms_norm_desc_init(C.byref(d), 0, 4096)
    assert lib.helix_rms_norm_grad_scratch_size(None, C.byref(d)) == 0
    lib.helix_rms_norm_desc_init(C.byref(d), 5, 16385)
    assert lib.helix_rms_norm_grad_scratch_size(None, C.byref(d)) == 0


def test_host_tensors_are_refused():
    torch = pytest.importorskip("torch")
    import helix_b200 as hx
    x, w = torch.ones(2, 8), torch.ones(8)
    for f in (lambda: hx.rms_norm(x, w), lambda: hx.quantize8(x), lambda: hx.matmul8(x, w, x, w),
              lambda: hx.gated_scan(x[None], x[None])):
        with pytest.raises(ValueError, match="CUDA"):
            f()
    with pytest.raises(AttributeError):
        hx.no_such_operator
