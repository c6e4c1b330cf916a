"""oracle/build_ref.py where the reference tree is missing."""
from oracle import build_ref


def test_without_the_reference_sources_nothing_is_built(tmp_path, monkeypatch):
    """No directory, or an empty one: the prebuilt library where there is one, else None."""
    lib = tmp_path / "lib.so"
    monkeypatch.setattr(build_ref, "LIB", str(lib))
    for root in (tmp_path / "absent", tmp_path):
        assert build_ref.build(str(root)) is None
    lib.touch()
    for root in (tmp_path / "absent", tmp_path):
        assert build_ref.build(str(root)) == str(lib)
