"""How the ragged steps' native binding is built and found, with the compiler
played by the test; and which streams the wrappers take."""
import os
import subprocess
import threading
import time
import types

import pytest
import torch

import spock_b200
from spock_b200 import builder


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A place of its own for the built file; the compiler writes there what `compiler.text` says, in two halves."""
    monkeypatch.setattr(builder, "HERE", str(tmp_path))
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "binding.cpp").write_text("// source")
    monkeypatch.setattr(builder, "CSRC", str(tmp_path / "csrc"))
    (tmp_path.parent / "include").mkdir(exist_ok=True)
    (tmp_path.parent / "include" / "spock_b200.h").write_text("// header")
    compiler = types.SimpleNamespace(text="whole", rc=0, runs=0, at_once=0, most=0, wrote=[])

    def run(cmd, **_):
        target = cmd[cmd.index("-o") + 1]
        compiler.runs += 1
        compiler.at_once += 1
        compiler.most = max(compiler.most, compiler.at_once)
        compiler.wrote.append(target)
        with open(target, "w") as f:
            f.write(compiler.text[:2])
            f.flush()
            time.sleep(0.1)
            assert not os.path.exists(builder.binding_path()) or open(builder.binding_path()).read() == "whole"
            if compiler.rc == 0:
                f.write(compiler.text[2:])
        compiler.at_once -= 1
        return subprocess.CompletedProcess(cmd, compiler.rc, "", "")

    monkeypatch.setattr(builder.subprocess, "run", run)
    return compiler


def test_binding_appears_whole(tree):
    path = builder.build_binding()
    assert path == builder.binding_path() and open(path).read() == "whole"
    assert path not in tree.wrote
    assert builder.build_binding() == path and tree.runs == 1  # nothing newer: not built again
    tree.rc = 1
    with pytest.raises(RuntimeError, match="g.. failed"):
        builder.build_binding(force=True)
    assert open(path).read() == "whole"  # a build that fails leaves what was there, and nothing beside it
    assert sorted(os.listdir(builder.HERE)) == sorted(["csrc", os.path.basename(path)])


def test_first_calls_at_once_build_it_once(tree):
    threads = [threading.Thread(target=builder.build_binding) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert tree.runs == 1 and tree.most == 1
    assert open(builder.binding_path()).read() == "whole"


def test_another_torch_has_a_binding_of_its_own(tree, monkeypatch):
    first = builder.build_binding()
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    second = builder.build_binding()
    assert first != second and tree.runs == 2 and os.path.exists(first)


def _unbuildable(*_, **__):
    raise RuntimeError("no compiler here")


def test_library_builds_without_the_binding(monkeypatch):
    monkeypatch.setattr(builder, "build", lambda force=False: "the library")
    monkeypatch.setattr(builder, "build_apps", lambda force=False: None)
    monkeypatch.setattr(builder, "build_binding", _unbuildable)
    with pytest.warns(UserWarning, match="no compiler here"):
        assert spock_b200.build() == "the library"


def test_wrappers_do_without_the_binding(monkeypatch):
    """A binding that cannot be had is said once and not tried again; None sends the wrappers their own way."""
    tried = []
    monkeypatch.setattr(spock_b200, "_BINDING", None)
    monkeypatch.setattr(builder, "build_binding", lambda *a, **k: tried.append(1) or _unbuildable())
    with pytest.warns(UserWarning, match="no compiler here"):
        assert spock_b200._binding() is None
    assert spock_b200._binding() is None and len(tried) == 1


def test_a_file_that_does_not_load_is_done_without(monkeypatch, tmp_path):
    broken = tmp_path / "_binding.so"
    broken.write_bytes(b"\x7fELF and no more")
    monkeypatch.setattr(spock_b200, "_BINDING", None)
    monkeypatch.setattr(builder, "build_binding", lambda *a, **k: str(broken))
    with pytest.warns(UserWarning):
        assert spock_b200._binding() is None


@pytest.mark.gpu
def test_calls_without_the_binding(cuda_ok, monkeypatch):
    from tests.test_gpu_ragged import DEV, F16, Cache, _gen, _i32
    g = _gen(2)
    c, s = Cache([70, 9], 16, 2, 64, F16, g), _i32([0, 3, 4])
    q = torch.randn(4, 8, 64, device=DEV, generator=g).half()
    with_it = spock_b200.paged_attention(q, s, *c.args(), 0.125)
    assert spock_b200._binding() is not None
    monkeypatch.setattr(spock_b200, "_BINDING", False)
    assert torch.equal(spock_b200.paged_attention(q, s, *c.args(), 0.125), with_it)


def test_streams_of_another_device_are_refused():
    stream = types.SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=77)
    assert spock_b200._stream_of(1, stream) == 77
    with pytest.raises(spock_b200.SpockError, match="stream: expected one of cuda:0") as e:
        spock_b200._stream_of(0, stream)
    assert e.value.code == spock_b200.SPOCK_ERR_INVALID
