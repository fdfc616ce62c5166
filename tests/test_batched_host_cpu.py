"""Host side of the batched operators without a GPU: sizes of scratch, a build where the binding's headers are missing,
and limits that Python and C share."""

import re
import sysconfig

from klab_b200 import _native, adapters, build, kv_pages


def test_plain_scratch_stays_small():
    """t and the projection in FP32 for 64 MiB of rows at a time, and the few behind the last part."""
    scratch = _native.lib().klab_adapter_scratch
    for wfmt in (_native.W_CBF16, _native.W_I8_G64):
        for m in (1, 300, 1169, 1185, 2048, 65535):
            assert 4 * min(m, 1024) * 14336 < scratch(wfmt, m, 14336, 4096, 16) <= 2 ** 26 + 2 ** 21
        # Rows that are each past a part's size: two tiles and the rest of a third.
        assert scratch(wfmt, 100, 2 ** 24, 64, 8) == 48 * 4 * (2 ** 24 + 8)


def test_build_without_python_headers(tmp_path, monkeypatch, capsys):
    """The library and the launcher are there, the binding is not, and an older one is taken away."""
    monkeypatch.setattr(build, "LAUNCHER", tmp_path / "bin" / "klab")
    monkeypatch.setattr(build, "BINDING", tmp_path / "klab_torch.so")
    monkeypatch.setattr(build, "OBJ", tmp_path)
    run, paths = build._run, sysconfig.get_paths()
    monkeypatch.setattr(build, "_compile", lambda source, headers, verbose=False: source)  # the library is not what this is about
    monkeypatch.setattr(build, "_run", lambda cmd: None if cmd[0] == build.nvcc() else run(cmd))
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {**paths, "include": str(tmp_path)})
    build.BINDING.write_bytes(b"of another torch")
    assert build.build() == build.LIBRARY
    assert build.LAUNCHER.exists() and not build.BINDING.exists()
    assert "Python.h" in capsys.readouterr().err


def test_limits_are_the_headers():
    header = (build.INCLUDE / "klab_b200.h").read_text()
    limits = {name: int(value) for name, value in re.findall(r"#define KLAB_((?:KV|ADAPTER)_MAX_\w+) (\d+)", header)}
    assert limits == {"KV_MAX_REQUESTS": kv_pages.MAX_REQUESTS, "KV_MAX_NEW": kv_pages.MAX_NEW,
                      "KV_MAX_GROUP": kv_pages.MAX_GROUP, "ADAPTER_MAX_RANK": adapters.MAX_RANK}
    steps = {name: int(value) for name, value in re.findall(r"#define KLAB_STEP_(\w+) (\d+)", header)}
    assert steps == {name[5:]: getattr(kv_pages, name) for name in dir(kv_pages) if name.startswith("STEP_")}
