"""Every test that is written is collected: a second definition of a name hides the first, and no run says so."""
import ast
import glob
import importlib
import os
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(HERE, "test_*.py"))), ids=os.path.basename)
def test_no_test_is_hidden_by_another(path):
    with open(path) as f:
        tree = ast.parse(f.read())
    written = {min([n.lineno] + [d.lineno for d in n.decorator_list]): n.name for n in tree.body if isinstance(n, ast.FunctionDef) and n.name.startswith("test")}
    if HERE not in sys.path:
        sys.path.insert(0, HERE)
    module = importlib.import_module(os.path.splitext(os.path.basename(path))[0])
    held = {v.__code__.co_firstlineno for name, v in vars(module).items() if name.startswith("test") and getattr(v, "__module__", None) == module.__name__ and hasattr(v, "__code__")}
    assert not {line: name for line, name in written.items() if line not in held}
