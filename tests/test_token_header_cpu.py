"""CPU check of the token operators' internal header: each function that it declares is defined with that many arguments."""
import os
import re
import subprocess

from gnnhwc import _cabi

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "channels-last-groupnorm_amd", "csrc", "gn_tokens.h")


def _arguments(text):
    """How many arguments a list has; commas inside brackets part none."""
    depth, n = 0, 1 if text.strip() else 0
    for c in text:
        depth += (c in "([<") - (c in ")]>")
        n += c == "," and depth == 0
    return n


def test_declared_functions_are_defined():
    text = open(HEADER).read().replace("\\\n", "")
    declared = {(name, _arguments(args)) for name, args in re.findall(r"^(?:\w+ )+(\w+)\((.*)\);$", text, flags=re.M)}
    for macro in re.findall(r"^#define GN_DECLARE_TOKENS\(S\)(.*)$", text, flags=re.M):
        for name, args in re.findall(r"hipError_t (\w+)##S\(((?:[^()]|\(&dw\))*)\);", macro + ";"):
            declared |= {(name + s, _arguments(args)) for s in re.findall(r"^GN_DECLARE_TOKENS\((\w+)\)", text, flags=re.M)}
    assert len(declared) >= 3 + 16
    symbols = subprocess.run(["nm", "-D", "--defined-only", "-C", _cabi.LIB_PATH], check=True, capture_output=True, text=True).stdout
    defined = {(name, _arguments(args)) for name, args in re.findall(r" T gn::(\w+)\((.*)\)$", symbols, flags=re.M)}
    assert declared <= defined, declared - defined
