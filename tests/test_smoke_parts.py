"""When smoke() may leave out the GPT step: only where its library cannot have
been built."""
import os

import __graft_entry__ as entry


def touch(*parts):
    path = os.path.join(*parts)
    os.makedirs(os.path.dirname(path), exist_ok=True)
    open(path, "w").close()


def test_gpt_step_is_expected_wherever_it_could_have_been_built(tmp_path, monkeypatch):
    monkeypatch.delenv("TEMPLIT_ROOT", raising=False)
    root = str(tmp_path / "checkout")
    os.makedirs(os.path.join(root, "templit_b200", "_build"))
    assert not entry.gpt_step_expected(root)
    # the headers: beside the repository, or where TEMPLIT_ROOT says
    touch(str(tmp_path), "reference", "include", "passes", "compile.h")
    assert entry.gpt_step_expected(root)
    monkeypatch.setenv("TEMPLIT_ROOT", str(tmp_path / "nowhere"))
    assert not entry.gpt_step_expected(root)
    touch(str(tmp_path), "elsewhere", "include", "passes", "compile.h")
    monkeypatch.setenv("TEMPLIT_ROOT", str(tmp_path / "elsewhere"))
    assert entry.gpt_step_expected(root)


def test_gpt_step_is_expected_beside_what_else_was_built(tmp_path, monkeypatch):
    monkeypatch.setenv("TEMPLIT_ROOT", str(tmp_path / "nowhere"))
    for made in ("libtemplit_gpt.so", "libtemplit_runtime.so", os.path.join("tests", "test_optimizer")):
        root = str(tmp_path / made.replace(os.sep, "_"))
        touch(root, "templit_b200", "_build", "libtemplit_cuda.so")
        assert not entry.gpt_step_expected(root)
        touch(root, "templit_b200", "_build", made)
        assert entry.gpt_step_expected(root)
