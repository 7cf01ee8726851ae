"""The block operators of a package that is loaded under another name, as
ComfyUI loads a folder of custom_nodes."""

import os
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

LOAD = """
import importlib, importlib.util, sys, torch
def load(name):
    path = %r
    spec = importlib.util.spec_from_file_location(name, path + "/__init__.py", submodule_search_locations=[path])
    sys.modules[name] = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(sys.modules[name])
    return importlib.import_module(name + ".vc_attention"), importlib.import_module(name + ".vc_attention._native")
""" % os.path.join(ROOT, "comfyui_vc_attention_b200")


def _python(body, cwd):
    """In a folder from which no package of the usual name can be imported."""
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    r = subprocess.run([sys.executable, "-c", LOAD + textwrap.dedent(body)], cwd=cwd, capture_output=True, text=True, env=env)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_copies_side_by_side(tmp_path):
    _python("""
        for name in ("copy_a", "copy_b"):
            vc, _ = load(name)
            plan = vc.packed_plan([4], heads=2, head_dim=64, device="cpu")
            try:
                vc.packed_attention(*[torch.zeros(1, 2, 4, 64)] * 3, plan)
                raise SystemExit("CPU tensors were taken")
            except RuntimeError as e:
                assert "CUDA" in str(e)
    """, str(tmp_path))


def test_a_foreign_object_is_no_plan(tmp_path):
    from comfyui_vc_attention_b200.vc_attention._host import host_ops
    import torch
    x = torch.zeros(1, 1, 4, 64)
    for bad in (None, 3, object()):
        with pytest.raises((TypeError, ValueError)):
            host_ops().packed_attention(x, x, x, bad, None, None)


@pytest.mark.gpu
def test_errors_are_those_of_the_loaded_copy(tmp_path):
    _python("""
        copies = [load("copy_a"), load("copy_b")]
        assert importlib.util.find_spec("comfyui_vc_attention_b200") is None
        assert copies[0][1].VCAttnError is not copies[1][1].VCAttnError
        for vc, native in copies + copies[:1]:
            native.inject_fault("vcattn_quantize_blocks")
            try:
                vc.quantize_blocks(torch.ones(4, 128, device="cuda"))
                raise SystemExit("the injected fault did not show")
            except native.VCAttnError as e:
                assert e.code == native.ERR_INJECTED and "injected" in str(e)
            finally:
                native.inject_fault(None)
    """, str(tmp_path))
