"""What a module's forward computes, read from its source as an expression of its parts.

A patcher that puts another forward in a module's place has to know the formula that it
replaces: that the parts have the usual names, or are called in the usual order, does not
say what else happens between them (a learned scale of a branch, stochastic depth, a
factor, a branch that reads another value, dropout). Only forwards without branches and
loops are read, of assignments to local names, calls of the module's parts, sums and
products of two values and the unpacking of a part's results; any other has no form, and
whoever asks leaves the module alone. Nothing is executed.
"""

from __future__ import annotations

import ast
import inspect
from typing import NamedTuple


class Form(NamedTuple):
    value: tuple         # what is returned
    calls: tuple         # names of the parts called, in order
    adds: int            # number of sums
    params: tuple        # names of the arguments without self
    var_kw: str | None   # name of the ** argument


def arg(name: str) -> tuple:
    return ("arg", name)


def call(part: str, *args, kwargs=None, star=None) -> tuple:
    """A part's result; star: the expression passed with **, or None."""
    return ("call", part, args, tuple(sorted((kwargs or {}).items())), star)


def item(index: int, count: int, value: tuple) -> tuple:
    """One of the results that a call is unpacked into."""
    return ("item", index, count, value)


def add(a: tuple, b: tuple) -> tuple:
    return ("add", *sorted((a, b), key=repr))


def mul(a: tuple, b: tuple) -> tuple:
    return ("mul", *sorted((a, b), key=repr))


class _NoForm(Exception):
    pass


class _Reader:
    def __init__(self, self_name: str, names):
        self.self_name, self.env = self_name, {n: arg(n) for n in names}
        self.calls, self.adds = [], 0

    def value(self, node) -> tuple:
        if isinstance(node, ast.Name) and node.id in self.env:
            return self.env[node.id]
        if isinstance(node, ast.BinOp) and isinstance(node.op, (ast.Add, ast.Mult)):
            a, b = self.value(node.left), self.value(node.right)
            if isinstance(node.op, ast.Mult):
                return mul(a, b)
            self.adds += 1
            return add(a, b)
        if isinstance(node, ast.Call) and isinstance(node.func, ast.Attribute) and \
                isinstance(node.func.value, ast.Name) and node.func.value.id == self.self_name:
            args = [self.value(a) for a in node.args]
            kwargs = {k.arg: self.value(k.value) for k in node.keywords}
            if len(kwargs) != len(node.keywords):  # (two with **)
                raise _NoForm
            self.calls.append(node.func.attr)
            return call(node.func.attr, *args, kwargs={k: v for k, v in kwargs.items() if k},
                        star=kwargs.get(None))
        raise _NoForm

    def assign(self, target, value: tuple) -> None:
        if isinstance(target, ast.Name) and target.id != self.self_name:
            self.env[target.id] = value
        elif isinstance(target, ast.Tuple) and value[0] == "call":
            for i, t in enumerate(target.elts):
                if not isinstance(t, ast.Name):
                    raise _NoForm
                self.assign(t, item(i, len(target.elts), value))
        else:
            raise _NoForm

    def run(self, body) -> tuple:
        """The value of the return that ends the body."""
        for node in body[:-1]:
            if isinstance(node, ast.Expr) and isinstance(node.value, ast.Constant):
                continue  # a docstring
            if not isinstance(node, ast.Assign):
                raise _NoForm
            value = self.value(node.value)
            for target in node.targets:
                self.assign(target, value)
        if not isinstance(body[-1], ast.Return) or body[-1].value is None:
            raise _NoForm
        return self.value(body[-1].value)


def form(fn) -> Form | None:
    """The form of a function (self first), None where it has none. The function is
    taken as it is: of one that wraps another, the wrapper is read."""
    code = getattr(fn, "__code__", None)
    if code is None:
        return None
    try:
        source = inspect.getsource(code)
        node = ast.parse("if True:\n" + source if source[0].isspace() else source).body[0]
    except (OSError, TypeError, SyntaxError, IndexError):
        return None
    if isinstance(node, ast.If):
        node = node.body[0]
    if not isinstance(node, ast.FunctionDef) or node.name != code.co_name:
        return None
    a = node.args
    if a.vararg or a.posonlyargs or not a.args:
        return None
    params = [p.arg for p in a.args[1:] + a.kwonlyargs]
    var_kw = a.kwarg.arg if a.kwarg else None
    reader = _Reader(a.args[0].arg, params + ([var_kw] if var_kw else []))
    try:
        value = reader.run(node.body)
    except _NoForm:
        return None
    return Form(value, tuple(reader.calls), reader.adds, tuple(params), var_kw)


def passed_on(f: Form, first: str) -> dict:
    """Keyword arguments of a call that hands on every argument but `first`, as it came."""
    return dict(kwargs={n: arg(n) for n in f.params if n != first},
                star=arg(f.var_kw) if f.var_kw else None)
