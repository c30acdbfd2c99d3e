"""Host-only parts of the operators that verify drafted tokens: tree masks,
refusals that need no device, and the layouts of the ABI's structs."""
import ctypes
import pathlib

import numpy as np
import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
LIB = ROOT / "raster-inference_amd" / "build" / "libdetgpu.so"
pytestmark = pytest.mark.skipif(not LIB.exists(), reason="libdetgpu.so not built")

rd = pytest.importorskip("rasterdet")


@pytest.mark.parametrize("parents,masks,depths", [
    ([], [], []),
    ([-1], [1], [0]),
    ([-1, 0, 1, 2], [1, 3, 7, 15], [0, 1, 2, 3]),
    ([-1, -1, 0, 0, 1, 4], [1, 2, 5, 9, 18, 50], [0, 0, 1, 1, 1, 2]),
    ([-1] + list(range(63)), [(1 << (i + 1)) - 1 for i in range(64)], list(range(64))),
])
def test_tree_masks(parents, masks, depths):
    m, d = rd.tree_masks(parents)
    assert m.tolist() == masks and d.tolist() == depths


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 2, 0], [-2], [-1] * 65])
def test_tree_masks_refuse_what_is_no_tree(parents):
    with pytest.raises(rd.DetError) as e:
        rd.tree_masks(parents)
    assert e.value.status == 1


def test_calls_without_a_context_are_refused():
    L = rd.lib()
    out = ctypes.c_void_p()
    assert L.det_rope_table_create(None, None, ctypes.byref(out)) == 1
    assert L.det_head_norm_rope(None, None, None, 1, 4, 0, None, 1) == 1
    assert L.det_attention_tree(None, None, None, 1, None, 1, None, None, 1, None, None, 1, 1, 1, None, 1) == 1
    assert L.det_adapters_create(None, 1, 1, None, 1, ctypes.byref(out)) == 1
    assert L.det_linear_adapters(None, None, None, 1, None, None, None) == 1
    assert L.det_select_tokens(None, None, 1, 1, 1, None, None, 1, None) == 1
    assert L.det_kv_view(None, None) == 1
    assert b"required" in L.det_ctx_last_error(None)
    for free in (L.det_rope_table_free, L.det_adapters_free):
        free(None)


def test_struct_sizes_match_the_header(tmp_path):
    import shutil
    import subprocess

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    names = {"det_rope_spec_t": rd.RopeSpec, "det_head_rows_t": rd.HeadRows, "det_attn_cache_t": rd.AttnCache,
             "det_adapter_spec_t": rd.AdapterSpec, "det_logit_rules_t": rd.LogitRules}
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "detgpu.h"\nint main(void) {' +
                   "".join(f'printf("%zu\\n", sizeof({n}));' for n in names) + "return 0; }\n")
    subprocess.run([cc, "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    sizes = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(s) for s in sizes] == [ctypes.sizeof(t) for t in names.values()]


def test_adapter_shapes_are_checked_before_the_upload():
    down, up = np.zeros((2, 8), dtype=np.int16), np.zeros((5, 2), dtype=np.int16)

    class NoContext:
        pass

    for bad in (rd.Adapter(down, up[:4]), rd.Adapter(down[:, :7], up), rd.Adapter(down, np.zeros((5, 3), np.int16)),
                rd.Adapter(down.astype(np.int8), up)):
        with pytest.raises(ValueError):
            rd.Adapters(NoContext(), 5, 8, [bad])
