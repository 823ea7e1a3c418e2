"""How baguanet.ops finds its built extension: the one that belongs to these
sources and flags, and never one that is still being written."""

import threading

import pytest

from baguanet import ops


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A tree of two sources and a header, whose extension is a text file: the
    header's text, which the compiler writes in two halves."""
    hip = tmp_path / "csrc" / "hip"
    hip.mkdir(parents=True)
    (tmp_path / "build" / "torch_ext").mkdir(parents=True)
    names = ("a.hip", "b.hip", "c.h")
    for n in names:
        (hip / n).write_text(n)
    monkeypatch.setattr(ops, "REPO_ROOT", tmp_path)
    monkeypatch.setattr(ops, "_sources", lambda: [hip / n for n in names[:2]])
    monkeypatch.setattr(ops, "_C", None)
    monkeypatch.setattr(ops, "_ERR", None)

    class Tree:
        lib = tmp_path / "build" / "torch_ext" / "baguanet_C.so"
        header = hip / "c.h"
        builds = 0
        half = lambda self: None  # called when half of it is written

        def compile(self, build_dir, sources, verbose, force):
            self.builds += 1
            text = self.header.read_text()
            with open(self.lib, "w") as f:
                f.write(text[:1])
                f.flush()
                self.half()
                f.write(text[1:])
            return self.lib.read_text()

        def load(self, **kw):
            """As in a process of its own."""
            ops._C = None
            return ops.build_extension(**kw)

    t = Tree()
    monkeypatch.setattr(ops, "_compile", t.compile)
    monkeypatch.setattr(ops, "_import_built", lambda lib: lib.read_text())
    return t


def test_built_once(tree):
    for _ in range(3):
        assert tree.load() == "c.h"
    assert tree.builds == 1
    assert tree.load(force=True) == "c.h" and tree.builds == 2
    assert ops.build_extension() == "c.h" and tree.builds == 2


def test_built_again_for_other_sources_flags_or_torch(tree, monkeypatch):
    assert tree.load() == "c.h"
    tree.header.write_text("other")
    assert tree.load() == "other" and tree.builds == 2
    monkeypatch.setattr(ops, "_HIP_FLAGS", ops._HIP_FLAGS + ["-g"])
    tree.load()
    assert tree.builds == 3
    monkeypatch.setenv("PYTORCH_ROCM_ARCH", "gfx942")
    tree.load()
    assert tree.builds == 4
    monkeypatch.setattr(ops.torch.version, "git_version", "another")
    tree.load()
    assert tree.builds == 5
    tree.load()
    assert tree.builds == 5


def test_time_stamps_do_not_count(tree):
    """Another checkout of the same sources is no reason to build."""
    tree.load()
    tree.header.touch()
    tree.load()
    assert tree.builds == 1


def test_not_loaded_half_written(tree):
    """A process that starts while another one links waits for it."""
    writing, go = threading.Event(), threading.Event()

    def half():
        writing.set()
        assert go.wait(20)

    tree.half = half
    results = []
    threads = [threading.Thread(target=lambda: results.append(tree.load()))
               for _ in range(2)]
    threads[0].start()
    assert writing.wait(20)
    threads[1].start()
    threads[1].join(0.3)
    assert not results  # neither has anything to load yet
    go.set()
    for t in threads:
        t.join(20)
    assert results == ["c.h", "c.h"] and tree.builds == 1


def test_broken_off_build_is_not_loaded(tree):
    def half():
        raise KeyboardInterrupt

    tree.load()
    tree.header.write_text("other")
    tree.half = half
    with pytest.raises(KeyboardInterrupt):
        tree.load()
    tree.half = lambda: None
    assert tree.load() == "other" and tree.builds == 3


def test_directory_that_cannot_be_written_to(tree, monkeypatch):
    tree.load()

    def refuse(self, *a, **kw):
        raise PermissionError(str(self))

    monkeypatch.setattr(type(tree.lib), "mkdir", refuse)
    assert tree.load() == "c.h" and tree.builds == 1


def test_file_system_without_locks(tree, monkeypatch):
    def refuse(file, how):
        raise OSError("no locks available")

    monkeypatch.setattr(ops.fcntl, "flock", refuse)
    assert tree.load() == "c.h" and tree.load() == "c.h" and tree.builds == 1


def test_loading_sets_no_architecture(tree, monkeypatch):
    monkeypatch.delenv("PYTORCH_ROCM_ARCH", raising=False)
    tree.load()
    tree.load()
    assert "PYTORCH_ROCM_ARCH" not in ops.os.environ and tree.builds == 1
