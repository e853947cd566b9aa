"""What `import pplb200` needs: the library.  torch is needed by calls on tensors, the compiled part of the binding by rotary positions, the
cache and attention."""
import os
import shutil
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "ppl.llm.kernel.cuda_b200")


def _python(code, path=PKG):
    done = subprocess.run([sys.executable, "-c", "import sys; sys.path.insert(0, %r)\n%s" % (path, code)], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    return done.stdout


def _without_binding(tmp_path):
    """The package with the library and no compiled part of the binding beside it."""
    shutil.copytree(os.path.join(PKG, "pplb200"), tmp_path / "pplb200", ignore=shutil.ignore_patterns("__pycache__"))
    (tmp_path / "lib").mkdir()
    os.symlink(os.path.join(PKG, "lib", "libpplb200_i8i8.so"), tmp_path / "lib" / "libpplb200_i8i8.so")
    return str(tmp_path)


def test_import_needs_no_torch():
    assert _python("""
sys.modules["torch"] = None  # importing it fails
import pplb200
assert "sm_100a" in pplb200.version() and pplb200.linear_workspace_bytes(16, 4096, 4096, pplb200.EPI_DEQUANT_F16) > 0
for name in ("RotaryTable", "attention", "kv_cache_write"):
    try:
        getattr(pplb200, name)
    except ImportError as e:
        print("torch" in str(e))
""").split() == ["True"] * 3


def test_import_loads_torch_only_where_it_is_used():
    _python("import pplb200\nassert 'torch' not in sys.modules and 'pplb200.attention' not in sys.modules")


def test_import_needs_no_binding(tmp_path):
    assert _python("""
import pplb200
assert "sm_100a" in pplb200.version() and pplb200.W8A8Linear and pplb200.minmax_quantize_fp16
try:
    pplb200.PagedKVCache
except ImportError as e:
    print("build.py" in str(e))
""", _without_binding(tmp_path)).split() == ["True"]


def test_names_of_attention():
    _python("""
import pplb200
names = ["PagedDecodeAttention", "PagedKVCache", "RotaryTable", "kv_cache_read", "kv_cache_write", "rotary_fp16", "rotary_kv_cache_write"]
assert set(names) <= set(dir(pplb200))
from pplb200 import RotaryTable, attention
assert RotaryTable is pplb200.RotaryTable is attention.RotaryTable and all(getattr(pplb200, n) is getattr(attention, n) for n in names)
assert all(n in vars(pplb200) for n in names)  # found at once from now on
try:
    pplb200.no_such_name
    sys.exit(1)
except AttributeError as e:
    assert "no_such_name" in str(e)
""")


def _build_module():
    import importlib.util
    spec = importlib.util.spec_from_file_location("pplb200_build_under_test", os.path.join(PKG, "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_another_torch_or_python_has_a_binding_of_its_own(monkeypatch):
    """The binding is compiled for one torch and one Python: it is built anew for others, and never loaded by them."""
    import torch
    import pplb200.attention
    build, commands = _build_module(), []
    here = build.binding_path()
    assert here == os.path.normpath(pplb200.attention.binding_path()) and os.path.exists(here) and torch.__version__ in here
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: commands.append(cmd))
    monkeypatch.setattr(build, "_stale", lambda target, deps: not os.path.exists(target))
    build.build()
    assert not commands
    monkeypatch.setattr(build, "torch_version", lambda: "99.1")
    build.build()
    assert len(commands) == 1 and build.binding_path() in commands[0] and build.binding_path() != here
    monkeypatch.setattr(torch, "__version__", "99.1")
    assert os.path.normpath(pplb200.attention.binding_path()) == build.binding_path()


def test_build_says_that_there_is_no_binding_without_torch(monkeypatch, capsys):
    build, commands = _build_module(), []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: commands.append(cmd))
    monkeypatch.setattr(build, "torch_home", lambda: None)
    monkeypatch.setattr(build, "_stale", lambda target, deps: not os.path.exists(target))
    assert build.build() == build.LIB and not commands
    assert "torch is not installed" in capsys.readouterr().out
