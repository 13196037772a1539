"""No module of the tests defines a name twice: the second definition of a test
takes the first one's place, which then no longer runs."""
import ast
import glob
import os

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
DEFINITIONS = (ast.FunctionDef, ast.AsyncFunctionDef, ast.ClassDef)


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(HERE, "*.py"))), ids=os.path.basename)
def test_names_are_defined_once(path):
    with open(path) as f:
        tree = ast.parse(f.read())
    for scope in [tree] + [n for n in tree.body if isinstance(n, ast.ClassDef)]:
        names = [n.name for n in scope.body if isinstance(n, DEFINITIONS)]
        twice = sorted({n for n in names if names.count(n) > 1})
        assert not twice, f"defined more than once: {', '.join(twice)}"
