"""CPU checks of __graft_entry__.py: what its script form runs, and that smoke() calls every operator it imports."""
import ast
import os
import types

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "__graft_entry__.py")


@pytest.fixture(scope="module")
def tree():
    return ast.parse(open(SOURCE).read())


def _main_block(tree):
    block, = [n for n in tree.body if isinstance(n, ast.If) and any(getattr(m, "id", None) == "__name__" for m in ast.walk(n.test))]
    return block


@pytest.mark.parametrize("words,calls", [([], ["build"]), (["smoke"], ["build", "smoke"])])
def test_the_script_builds_and_tests_on_request_and_does_nothing_else(words, calls, tree):
    ran = []
    names = {"build": lambda: ran.append("build"), "smoke": lambda: ran.append("smoke"), "sys": types.SimpleNamespace(argv=[SOURCE] + words)}
    exec(compile(ast.Module(_main_block(tree).body, []), SOURCE, "exec"), names)
    assert ran == calls


def test_smoke_calls_every_operator_that_it_imports(tree):
    smoke, = [n for n in tree.body if isinstance(n, ast.FunctionDef) and n.name == "smoke"]
    imported = {a.asname or a.name for n in ast.walk(smoke) if isinstance(n, ast.ImportFrom) and n.module == "gnnhwc" for a in n.names}
    called = {n.func.id for n in ast.walk(smoke) if isinstance(n, ast.Call) and isinstance(n.func, ast.Name)}
    assert {"window_attention", "window_attention_cached", "dropout"} <= imported and imported <= called
