"""Host side of the decode operators, without a GPU: devices and builds."""

import types

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def device_three(monkeypatch):
    """A process whose current CUDA device is 3 (of which only the index is asked); the devices of the workspaces made."""
    from heatvit_b200 import decode
    made = []
    stream = types.SimpleNamespace(synchronize=lambda: None)
    cuda = types.SimpleNamespace(current_device=lambda: 3, current_stream=lambda device: stream)
    monkeypatch.setattr(decode, "_torch", lambda: types.SimpleNamespace(cuda=cuda, device=torch.device))
    monkeypatch.setattr(decode, "_load", lambda: types.SimpleNamespace(attention_workspace=made.append))
    return made


@pytest.mark.parametrize("device,index", [(None, 3), ("cuda", 3), (torch.device("cuda"), 3), ("cuda:0", 0),
                                          (torch.device("cuda", 5), 5)])
def test_workspace_lives_on_the_device_that_was_meant(device_three, device, index):
    """A device without an index is the current one, as everywhere in torch."""
    from heatvit_b200 import decode
    ws = decode.AttentionWorkspace(device)
    assert device_three == [index] and ws.device == torch.device("cuda", index)


def test_workspace_refuses_what_is_no_cuda_device(device_three):
    from heatvit_b200 import decode
    with pytest.raises(ValueError, match="CUDA"):
        decode.AttentionWorkspace("cpu")
    assert device_three == []


def test_quantized_weight_keeps_no_graph(monkeypatch):
    """A parameter's e4m3 form is a plain tensor: it neither asks for gradients nor holds the float32 copies."""
    from heatvit_b200 import decode
    monkeypatch.setattr(decode, "_torch", lambda: torch)
    weight = torch.nn.Parameter(torch.randn(200, 150))
    q, scale = decode.quantize_weight_fp8(weight)
    assert not q.requires_grad and q.grad_fn is None and q._base.grad_fn is None
    assert not scale.requires_grad and scale.grad_fn is None
    plain, its_scale = decode.quantize_weight_fp8(weight.detach())
    assert torch.equal(q.view(torch.uint8), plain.view(torch.uint8)) and torch.equal(scale, its_scale)


# ---- builds -------------------------------------------------------------------------

def test_library_builds_without_torch(monkeypatch, tmp_path, capsys):
    """The C library needs nvcc alone: without torch the Python module is left out, and that is said."""
    import importlib.util
    from heatvit_b200 import build
    build.build()
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setattr(build, "NATIVE", str(tmp_path / "_decode_native.so"))
    assert build.build() == build.LIB
    assert not (tmp_path / "_decode_native.so").exists()
    assert "torch" in capsys.readouterr().err
    assert build.build_native(force=True) is None


def test_module_is_stale_beside_another_torch(monkeypatch, tmp_path):
    """The module uses torch's C++ interfaces, which other versions of torch or Python do not keep."""
    from heatvit_b200 import build
    build.build()
    assert build.native_up_to_date()
    with monkeypatch.context() as m:
        m.setattr(build, "native_made_for", lambda: "another torch")
        assert not build.native_up_to_date()
    assert build.native_up_to_date()
    made_for = build.native_made_for()
    assert torch.__version__ in made_for and build.sysconfig.get_config_var("EXT_SUFFIX") in made_for
