"""The V hooks (vtl_b200/vglue) read as text, since no V toolchain is at hand: what a compiler, or a leak, would show."""
import glob
import os
import re

import pytest

VGLUE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vtl_b200", "vglue")
HOOKS = [f for f in sorted(glob.glob(os.path.join(VGLUE, "*_d_b200.v"))) if os.path.basename(f) != "c_d_b200.v"]
FALLIBLE = r"\bs\.(?:as_tensor|upload|alloc|alloc_f32|resident|to_host)\("


def code(path):
    return re.sub(r"//[^\n]*", "", open(path).read())


def functions(path):
    """(name, signature, body) of each function of a file."""
    src = code(path)
    for m in re.finditer(r"^(?:pub )?fn (?:\([^)]*\) )?(\w+)\([^\n]*\{$", src, re.M):
        end = src.index("\n}", m.end())
        yield m.group(1), m.group(0), src[m.end():end]


def call_end(text, start):
    """The index behind the parenthesis that closes the one in front of `start`."""
    depth = 1
    for i in range(start, len(text)):
        depth += {"(": 1, ")": -1}.get(text[i], 0)
        if depth == 0:
            return i + 1
    raise AssertionError("unbalanced parentheses")


def test_there_are_hooks():
    names = {n for f in HOOKS for n, _, _ in functions(f)}
    assert {"linear_forward_f32", "embedding_backward_f32", "groupnorm_forward_f32", "dropout_forward_f32"} <= names


@pytest.mark.parametrize("path", HOOKS, ids=os.path.basename)
def test_results_are_unwrapped(path):
    """A call that may fail gives its value by `!`; only `return s.as_tensor(...)` of a function that returns one result
    hands the result on as it is."""
    for name, signature, body in functions(path):
        for m in re.finditer(FALLIBLE, body):
            end = call_end(body, m.end())
            if body[end:end + 1] == "!":
                continue
            line = body[body.rfind("\n", 0, m.start()) + 1:body.find("\n", end) if "\n" in body[end:] else len(body)]
            assert re.fullmatch(r"\s*return s\.as_tensor\(.*\)", line, re.S), (name, line)
            assert re.search(r"\) !&vtl\.Tensor\[f32\] \{$", signature), name


# what a hook hands on to its caller instead of freeing it: the indices that the pooling's backward call frees, the codes of
# a quantised layer
HANDED_ON = {("maxpool2d_forward_f32", "didx"), ("new_quant_linear", "d_wq"), ("new_quant_linear", "d_sw")}


@pytest.mark.parametrize("path", [f for f in HOOKS if "session" not in f], ids=os.path.basename)
def test_buffers_are_freed(path):
    """as_tensor copies to the host and takes nothing over: whatever a hook allocates or uploads it frees in a defer."""
    for name, _, body in functions(path):
        freed = set()
        for m in re.finditer(r"\bdefer \{(.*?)\n\t\}", body, re.S):
            block = m.group(1)
            freed |= set(re.findall(r"s\.free\((\w+)\)", block))
            for names in re.findall(r"for \w+ in \[([^\]]*)\]", block):
                freed |= {n.strip() for n in names.split(",")}
        for line in body.splitlines():
            m = re.match(r"\s*([\w, ]+?) := (.*\bs\.(?:alloc|alloc_f32|upload)\(.*)", line)
            if m:
                for var in m.group(1).split(","):
                    assert var.strip() in freed or (name, var.strip()) in HANDED_ON, (name, var.strip())


@pytest.mark.parametrize("path", HOOKS, ids=os.path.basename)
def test_sizes_in_bytes_are_no_products_of_ints(path):
    """An int holds less than 2 GiB: 2^30 elements of four bytes would come to no bytes at all.  Sizes are counted by alloc_f32,
    from dimensions, or in usize."""
    src = code(path)
    for m in re.finditer(r"\bs\.alloc\(", src):
        args = src[m.end():call_end(src, m.end()) - 1]
        assert "*" not in args or all(f.strip().startswith("usize(") for f in args.split("*")) or args == "bytes", args
    for m in re.finditer(r"usize\(", src):
        args = src[m.end():call_end(src, m.end()) - 1]
        assert not re.search(r"\*\s*4\b|\b4\s*\*", args), args
    if path.endswith("session_d_b200.v"):
        assert "pub fn (s &DeviceSession) alloc(bytes usize) !voidptr {" in src
        assert "pub fn (s &DeviceSession) alloc_f32(dims ...int) !voidptr {" in src
        total = src[src.index(") alloc_f32("):]
        assert "usize(4)" in total and "*= usize(dim)" in total


def test_group_norm_takes_any_rank():
    """[batch, channels] and [batch, ..., channels]: no hook of group norm indexes a fixed third dimension."""
    path = os.path.join(VGLUE, "token_layers_d_b200.v")
    bodies = {n: b for n, _, b in functions(path)}
    for name in ("groupnorm_forward_f32", "groupnorm_backward_f32"):
        assert "shape[2]" not in bodies[name] and "shape[1]" not in bodies[name], name
        assert "norm_sizes(x.shape)!" in bodies[name], name
    body = bodies["norm_sizes"]
    assert "shape.len < 2" in body and "return error(" in body and "shape.last()" in body and "shape[1..shape.len - 1]" in body


@pytest.mark.parametrize("path", HOOKS, ids=os.path.basename)
def test_no_field_has_the_name_of_a_method(path):
    src = code(path)
    for m in re.finditer(r"struct (\w+) \{(.*?)\n\}", src, re.S):
        fields = set(re.findall(r"^\t(\w+)\s+\S", m.group(2), re.M))
        methods = set(re.findall(r"fn \((?:mut )?\w+ &?%s\) (\w+)\(" % m.group(1), src))
        assert not fields & methods, (m.group(1), fields & methods)
