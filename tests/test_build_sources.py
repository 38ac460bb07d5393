"""CPU: the kernel sources are what the build reads, and profiles are tied to the sources that they were measured on."""
import os

from ai2bmd_amd import build


def test_every_kernel_source_is_built():
    listed = {f for f in build.SOURCES + build.HEADERS if os.sep not in f}
    assert set(os.listdir(build.CSRC)) == listed


def test_an_engine_profile_outlives_changes_of_the_layer_operators(tmp_path, monkeypatch):
    """bench.py reports a committed profile's traffic while the engine's sources are those measured, whatever becomes of the
    layer operators beside it - and no longer once an engine source, or the engine's part of vsn.h, changes"""
    import json
    import shutil

    import bench

    csrc = tmp_path / "ai2bmd_amd" / "csrc"
    shutil.copytree(build.CSRC, csrc)
    shutil.copytree(os.path.join(build.CSRC, "..", "..", "include"), tmp_path / "include")
    monkeypatch.setattr(build, "CSRC", str(csrc))
    profile = tmp_path / "traffic.json"
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    monkeypatch.setattr(bench, "TRAFFIC_PROFILE", profile.name)
    profile.write_text(json.dumps({"build_digest": build._digest(engine_only=True), "chig_md": {"k": 53.7e6},
                                   "kernel_ns": {"chig_md": {"k": {"avg_ns": 1.0}}}}))
    reported = lambda: (bench.traffic_from_profile("chig_md", "k")[0], bench.rocprof_from_profile("chig_md", "k"))
    present = (53.7e6, {"avg_ns": 1.0})
    assert reported() == present

    def change(path, old, new):
        text = path.read_text()
        assert old in text
        path.write_text(text.replace(old, new, 1))

    whole = build._digest()
    change(csrc / "attention.h", "kTile = 32;", "kTile = 32; ")
    change(csrc / "norm.hip", "namespace vsn {", "namespace vsn { ")
    change(tmp_path / "include" / "vsn.h", "int vsn_layernorm(int device_id,", "int vsn_layernorm(int  device_id,")
    assert build._digest() != whole and reported() == present
    header = (tmp_path / "include" / "vsn.h").read_text()
    change(tmp_path / "include" / "vsn.h", "int vsn_hopt_run(", "int  vsn_hopt_run(")
    assert reported() == (None, None)
    (tmp_path / "include" / "vsn.h").write_text(header)
    assert reported() == present
    change(csrc / "gemm.hip", "namespace vsn {", "namespace vsn { ")
    assert reported() == (None, None)


def test_the_layer_files_are_of_the_build():
    assert set(build.LAYER_FILES) <= set(build.SOURCES + build.HEADERS)
