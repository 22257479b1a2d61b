"""CPU: a variant library holds every source of the library, the ones with flags of their own among them."""
from opensplat_amd import _build


def test_a_variant_is_built_from_all_sources(monkeypatch):
    runs = []
    monkeypatch.setattr(_build, "_run", runs.append)
    target = _build.build_variant("other", ["-DSOMETHING=1"])
    assert target.endswith("libgsplat_hip_other.so") and target != _build.HIP_LIB
    assert all("-DSOMETHING=1" in r for r in runs)
    *plain, link = runs
    objects = [r[r.index("-o") + 1] for r in plain]
    assert [r[r.index("-c") + 1] for r in plain] == _build.HIP_SOURCES_PLAIN
    assert all(f in r for r in plain for f in _build.HIPCC_PLAIN_FLAGS)
    assert all(o in link for o in objects) and all(s in link for s in _build.HIP_SOURCES) and link[-1] == target
    # the library's own objects are not overwritten
    assert not set(objects) & {s.replace(".hip", ".o") for s in _build.HIP_SOURCES_PLAIN}
    assert "-shared" in link and not any("-shared" in r for r in plain)


def test_the_script_goes_through_it():
    import os

    script = open(os.path.join(_build.ROOT, "scripts", "build_variant.sh")).read()
    assert "_build.build_variant(" in script and ".hip" not in script.replace("libgsplat_hip", "").replace("hipcc", "")
