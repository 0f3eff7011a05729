"""The in-tree extension must link (no undefined symbols) and expose the full kernel API."""


def test_extension_imports_and_exports():
    from pytorch_cifar_amd import _native

    C = _native.lib()
    for name in ["conv_fwd", "conv_dgrad", "conv_wgrad", "weight_prep", "bn_stats", "bn_finalize",
                 "bn_apply", "bn_backward", "augment", "gap_fwd", "gap_bwd", "avgpool_fwd",
                 "maxpool_fwd", "ce_fused", "sgd_step", "se_scale_fwd", "dw_fwd", "dw_dgrad",
                 "dw_wgrad", "direct_fwd", "direct_dgrad", "direct_wgrad", "RcclComm",
                 "rccl_unique_id", "set_conv_tile"]:
        assert hasattr(C, name), name


def test_other_flags_are_another_build(tmp_path, monkeypatch):
    """Objects and the library are of their sources and of the command that compiled them."""
    import os

    from pytorch_cifar_amd import _build

    src, obj = tmp_path / "k.hip", tmp_path / "k.hip.o"
    src.write_text("")
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        obj.write_text("")
        return type("R", (), {"returncode": int("bad" in cmd), "stderr": ""})

    monkeypatch.setattr(_build.subprocess, "run", run)
    need = lambda flags: _build._needs_build(str(src), str(obj), [], flags)   # noqa: E731
    assert need(["-O3"])
    _build._compile(str(src), str(obj), ["-O3"], False)
    assert "-packed-fp32-ops" in runs[0]
    assert not need(["-O3"]) and need(["-O2"])
    digest = _build.source_digest()
    with monkeypatch.context() as m:
        m.setattr(_build, "NO_PACKED_FP32", [])
        assert need(["-O3"]) and _build.source_digest() != digest
    assert not need(["-O3"]) and _build.source_digest() == digest
    os.utime(src, (os.path.getmtime(obj) + 5,) * 2)
    assert need(["-O3"])
    os.utime(src, (0, 0))
    assert not need(["-O3"])
    # a compile that failed leaves nothing that looks built
    try:
        _build._compile(str(src), str(obj), ["bad"], False)
    except RuntimeError:
        pass
    assert need(["-O3"]) and need(["bad"])
