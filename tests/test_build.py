"""The build's own steps, with stand-ins for the compilers: which files are left after which failure."""
import os

import pytest

from experts4bit_qlora_amd import _build as B

WRITES = '#!/bin/sh\nwhile [ $# -gt 0 ]; do if [ "$1" = -o ]; then echo new > "$2"; fi; shift; done\n'
FAILS = "#!/bin/sh\necho no such header >&2\nexit 1\n"


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """An older library and binding in place; tools(hipcc, cxx) sets the compilers' stand-ins."""
    out, binding = tmp_path / "libe4b_amd.so", tmp_path / "libe4b_torch.so"
    out.write_text("old\n"), binding.write_text("old\n")
    monkeypatch.setattr(B, "OUT", str(out))
    monkeypatch.setattr(B, "TORCH_OUT", str(binding))

    def tools(hipcc, cxx):
        for name, text in (("HIPCC", hipcc), ("CXX", cxx)):
            path = tmp_path / name
            path.write_text(text)
            path.chmod(0o755)
            monkeypatch.setenv(name, str(path))

    def left():
        assert not [f for f in os.listdir(tmp_path) if f.endswith(".tmp")]
        return [f.read_text().strip() if f.exists() else None for f in (out, binding)]

    return tools, left


def test_both_are_built(tree):
    tools, left = tree
    tools(WRITES, WRITES)
    B.build()
    assert left() == ["new", "new"]


def test_the_library_needs_hipcc_alone(tree):
    """Where the binding does not compile, the library is there all the same, and no binding of an older one."""
    tools, left = tree
    tools(WRITES, FAILS)
    with pytest.raises(RuntimeError, match="no such header"):
        B.build()
    assert left() == ["new", None]


def test_the_library_needs_no_torch_headers(tree, monkeypatch):
    tools, left = tree
    tools(WRITES, WRITES)

    def missing(*a):
        raise ImportError("no torch")

    monkeypatch.setattr(B, "_torch_commands", missing)
    with pytest.raises(RuntimeError, match="no torch"):
        B.build()
    assert left() == ["new", None]


def test_a_link_of_the_binding_that_fails(tree):
    tools, left = tree
    tools(WRITES, '#!/bin/sh\ncase "$*" in *-shared*) exit 1;; esac\n' + WRITES.partition("\n")[2])
    with pytest.raises(RuntimeError, match="CXX failed"):
        B.build()
    assert left() == ["new", None]


def test_the_library_by_itself(tree):
    tools, left = tree
    tools(WRITES, FAILS)
    B.build(binding=False)
    assert left() == ["new", None]


def test_a_library_that_does_not_compile_leaves_everything(tree):
    tools, left = tree
    tools(FAILS, WRITES)
    with pytest.raises(RuntimeError, match="HIPCC failed"):
        B.build()
    assert left() == ["old", "old"]
