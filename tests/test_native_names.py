"""No function of the package's modules replaces another of the same module."""
from __future__ import annotations

import ast
import glob
import os

import pytest

import neural_shift_cuda_amd

ROOT = os.path.dirname(neural_shift_cuda_amd.__file__)


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(ROOT, "**", "*.py"),
                                                  recursive=True)),
                         ids=lambda p: os.path.relpath(p, ROOT))
def test_names_are_defined_once(path):
    def names(body):
        return [n.name for n in body if isinstance(n, (ast.FunctionDef, ast.ClassDef))]

    tree = ast.parse(open(path).read())
    bodies = [tree.body] + [n.body for n in ast.walk(tree) if isinstance(n, ast.ClassDef)]
    for body in bodies:
        seen = names(body)
        assert len(seen) == len(set(seen)), sorted(n for n in seen if seen.count(n) > 1)
