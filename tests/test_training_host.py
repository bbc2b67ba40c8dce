"""The Python layer of the training operators, without a GPU."""
import pytest


@pytest.fixture
def training():
    import __graft_entry__
    __graft_entry__.build()
    from aethelstream_b200 import training
    return training


def test_workspace_sizes_are_kept_per_device(training, monkeypatch):
    """Two devices with different numbers of SMs, in turn: each gets its own size."""
    current, asked = [0], []

    class Library:
        @staticmethod
        def aeth_cut_ce_workspace(n, d, vocab, backward, size):
            asked.append((n, d, vocab, backward))
            size._obj.value = (7, 148)[current[0]] * n
            return 0

    monkeypatch.setattr(training, "_lib", Library)
    training._workspace_bytes.cache_clear()
    try:
        for dev, want in ((0, 70), (1, 1480), (0, 70), (1, 1480)):
            current[0] = dev
            assert training._workspace_bytes("aeth_cut_ce_workspace", dev, 10, 64, 100, 0) == want
        assert asked == [(10, 64, 100, 0)] * 2
    finally:
        training._workspace_bytes.cache_clear()


def test_scales_without_dimensions_are_refused(training):
    """One row of one block: as many scales as are due, but not in the checkpoint's shape."""
    import torch
    ck = training.ActivationCheckpoint(torch.zeros(1, 64, dtype=torch.int8), torch.ones(()), torch.bfloat16)
    with pytest.raises(ValueError, match="ActivationCheckpoint"):
        training._ckpt_args("checkpoint_decode", ck, -1)


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """build.py on two small units and a compiler that writes down its flags; it
    stops half-way while the file `stop` is there."""
    import stat

    import __graft_entry__
    mod = __graft_entry__._load_builder()
    src = tmp_path / "csrc"
    src.mkdir()
    for u in ("a", "b"):
        (src / f"{u}.cu").write_text("")
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "aeth_galore.h").write_text("")
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(f"""#!/bin/sh
out=; ins=; flags=; prev=
for x in "$@"; do
  case "$prev" in -o) out=$x;; esac
  case "$x" in -D*) flags="$flags $x";; *.o) ins="$ins $x";; esac
  prev=$x
done
case " $* " in
  *" -shared "*) cat $ins > "$out";;
  *) printf half > "$out"; [ -e {tmp_path}/stop ] && exit 1; echo "whole$flags" > "$out";;
esac
""")
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("NVCC", str(nvcc))
    for name, value in (("CSRC", str(src)), ("LIB", str(tmp_path / "lib.so")), ("OBJ", str(tmp_path / "_obj")),
                        ("UNITS", ("a", "b")), ("ROOT", str(tmp_path))):
        monkeypatch.setattr(mod, name, value)
    return mod


def test_a_build_that_stopped_leaves_no_object_behind(builder, tmp_path):
    (tmp_path / "stop").write_text("")
    with pytest.raises(RuntimeError):
        builder.build()
    (tmp_path / "stop").unlink()
    builder.build()
    assert (tmp_path / "lib.so").read_text() == "whole\nwhole\n"


def test_flags_of_one_build_stay_out_of_the_next(builder, tmp_path):
    import os
    builder.build(force=True, extra=["-DX"])
    assert (tmp_path / "lib.so").read_text() == "whole -DX\nwhole -DX\n"
    after = os.path.getmtime(tmp_path / "lib.so") + 10
    os.utime(tmp_path / "csrc" / "a.cu", (after, after))
    builder.build()
    assert (tmp_path / "lib.so").read_text() == "whole\nwhole\n"
