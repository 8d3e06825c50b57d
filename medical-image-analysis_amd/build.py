"""Builds libmia_hip.so (hand-written gfx950 kernels + C ABI) in-tree with hipcc.

hipcc cross-compiles for gfx950 without a GPU, so this runs in the build container; the .so travels to
the GPU box with the source tree.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmia_hip.so")
# No packed-fp32 instructions (v_pk_add/mul/fma_f32): hipcc forms them by itself from ordinary float code at -O3, and some
# of their forms have given wrong results now and then, without an error. The host pass warns that it does not know the
# feature, which is harmless.
HIPFLAGS = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
SOURCES = ["runtime.hip", "gemm.hip", "dwconv.hip", "pointwise.hip", "head.hip", "preprocess.hip", "optim.hip", "seg.hip", "metrics.hip", "augment.hip", "blocknorm.hip", "relpos.hip"]


def kernel_tree_hash() -> str:
    """Digest of everything that decides which kernels a training step launches and what they move: the kernel
    sources and the Python modules that sequence them. Measurements kept on file (HBM traffic per kernel from the
    counter passes) carry the digest of the tree they were taken on, so a reader can tell whether they still apply."""
    import hashlib
    h = hashlib.sha256()
    files = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hip", ".h")))
    files += [os.path.join(HERE, f) for f in ("ops.py", "trunk.py", "head_ops.py", "heads.py", "optim.py", "ddp.py")]
    for path in files:
        h.update(os.path.basename(path).encode())
        with open(path, "rb") as f:
            h.update(f.read())
    return h.hexdigest()[:16]


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    # the public header too: _lib.py derives every ctypes prototype from it, so a library older than the header
    # could be called with the wrong argument list
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "mia_hip.h"), __file__]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = True) -> str:
    if not force and not _stale():
        return LIB
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    objs = []
    procs = []
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    for src in SOURCES:
        path = os.path.join(CSRC, src)
        if not os.path.exists(path):
            continue
        obj = os.path.join(HERE, "build", src.replace(".hip", ".o"))
        objs.append(obj)
        if (not force) and os.path.exists(obj) and os.path.getmtime(obj) > max(
                os.path.getmtime(path), os.path.getmtime(os.path.join(CSRC, "common.h")), os.path.getmtime(__file__)):
            continue
        cmd = [hipcc, *HIPFLAGS, "-c", path, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd)))
    for src, p in procs:
        if p.wait() != 0:
            raise RuntimeError(f"hipcc failed on {src}")
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return LIB


# ------------------------------------------------------------------------------------------------
# Fast-call binding. A training step makes ~870 calls into the library; through ctypes each costs ~5 us of argument
# conversion on the host, a fifth of the step's enqueue time. The module generated here has one METH_FASTCALL
# wrapper per entry point of include/mia_hip.h: it converts ints / floats / addresses straight from the argument
# vector and calls the function through a pointer the loader hands over (the SAME loaded libmia_hip.so that ctypes
# opened, so there is one copy of the library's state). Purely a faster way to make the same calls: _lib.py uses it when
# it is present and was generated from the same prototypes, and the ctypes binding otherwise.
# ------------------------------------------------------------------------------------------------
def _load_proto():
    import importlib.util
    spec = importlib.util.spec_from_file_location("mia_proto", os.path.join(HERE, "_proto.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def fast_module_path() -> str:
    import sysconfig
    return os.path.join(HERE, "_mia_fast" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))


_CONV = {
    "int": ("int", "(int)PyLong_AsLong(args[{i}])"),
    "longlong": ("long long", "PyLong_AsLongLong(args[{i}])"),
    "ulonglong": ("unsigned long long", "PyLong_AsUnsignedLongLongMask(args[{i}])"),
    "float": ("float", "(float)PyFloat_AsDouble(args[{i}])"),
    "double": ("double", "PyFloat_AsDouble(args[{i}])"),
    "ptr": ("void*", "as_ptr(args[{i}])"),
}


def generate_fast_source() -> str:
    proto = _load_proto()
    protos = proto.parse_protos()
    names = [n for n in sorted(protos) if protos[n][0] in ("int", "longlong")]
    out = ['/* generated by build.py from include/mia_hip.h -- do not edit */',
           '#define PY_SSIZE_T_CLEAN', '#include <Python.h>', '',
           f'static const char* DIGEST = "{proto.header_digest()}";',
           f'static void* FN[{len(names)}];', 'static PyObject* ERR = NULL;',
           'static const char* (*LAST_ERROR)(void) = NULL;', '',
           '/* an address: int, None, a ctypes pointer object (its .value) or a ctypes array / buffer (its address) */',
           'static void* as_ptr(PyObject* o) {',
           '    if (o == Py_None) return NULL;',
           '    if (PyLong_Check(o)) return PyLong_AsVoidPtr(o);',
           '    PyObject* v = PyObject_GetAttrString(o, "value");',
           '    if (v) {',
           '        void* p = v == Py_None ? NULL : PyLong_AsVoidPtr(v);',
           '        Py_DECREF(v);',
           '        return p;',
           '    }',
           '    PyErr_Clear();',
           '    Py_buffer b;',
           '    if (PyObject_GetBuffer(o, &b, PyBUF_SIMPLE) == 0) {',
           '        void* p = b.buf;',
           '        PyBuffer_Release(&b);',
           '        return p;',
           '    }',
           '    return NULL;   /* the error set by GetBuffer is reported by the caller */',
           '}', '']
    for idx, n in enumerate(names):
        ret, kinds = protos[n]
        cret = "int" if ret == "int" else "long long"
        ctypes_ = ", ".join(_CONV[k][0] for k in kinds) or "void"
        out.append(f'static PyObject* w_{n}(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {{')
        out.append(f'    if (nargs != {len(kinds)}) {{ PyErr_Format(PyExc_TypeError, "{n} takes {len(kinds)} arguments (%zd given)", nargs); return NULL; }}')
        out.append(f'    if (!FN[{idx}]) {{ PyErr_SetString(PyExc_RuntimeError, "{n}: binding not initialised"); return NULL; }}')
        for i, k in enumerate(kinds):
            out.append(f'    {_CONV[k][0]} a{i} = {_CONV[k][1].format(i=i)};')
        out.append('    if (PyErr_Occurred()) return NULL;')
        call = f'(({cret} (*)({ctypes_}))FN[{idx}])({", ".join(f"a{i}" for i in range(len(kinds)))})'
        out.append(f'    {cret} rc = {call};')
        if ret == "int" and n not in proto.COUNTS:
            out.append('    if (rc != 0) {')
            out.append(f'        PyErr_Format(ERR ? ERR : PyExc_RuntimeError, "{n} failed (%d): %s", rc, LAST_ERROR ? LAST_ERROR() : "?");')
            out.append('        return NULL;')
            out.append('    }')
        out.append('    return PyLong_FromLong((long)rc);' if ret == "int" else '    return PyLong_FromLongLong(rc);')
        out.append('}')
        out.append('')
    out += ['/* bind({name: address}, error class, address of mia_last_error) */',
            'static PyObject* w_bind(PyObject* self, PyObject* a) {',
            '    PyObject *table, *err; unsigned long long last;',
            '    if (!PyArg_ParseTuple(a, "OOK", &table, &err, &last)) return NULL;',
            '    static const char* NAMES[] = {' + ", ".join(f'"{n}"' for n in names) + '};',
            f'    for (int i = 0; i < {len(names)}; ++i) {{',
            '        PyObject* v = PyDict_GetItemString(table, NAMES[i]);',
            '        if (!v) { PyErr_Format(PyExc_KeyError, "no address for %s", NAMES[i]); return NULL; }',
            '        FN[i] = PyLong_AsVoidPtr(v);',
            '        if (PyErr_Occurred()) return NULL;',
            '    }',
            '    Py_XDECREF(ERR); ERR = err; Py_INCREF(ERR);',
            '    LAST_ERROR = (const char* (*)(void))(size_t)last;',
            '    Py_RETURN_NONE;',
            '}',
            'static PyObject* w_digest(PyObject* self, PyObject* a) { return PyUnicode_FromString(DIGEST); }', '',
            'static PyMethodDef METHODS[] = {']
    for n in names:
        out.append(f'    {{"{n}", (PyCFunction)(void (*)(void))w_{n}, METH_FASTCALL, NULL}},')
    out += ['    {"bind", w_bind, METH_VARARGS, NULL},', '    {"digest", w_digest, METH_NOARGS, NULL},',
            '    {NULL, NULL, 0, NULL}};',
            'static struct PyModuleDef MOD = {PyModuleDef_HEAD_INIT, "_mia_fast", NULL, -1, METHODS};',
            'PyMODINIT_FUNC PyInit__mia_fast(void) { return PyModule_Create(&MOD); }', '']
    return "\n".join(out)


def build_fast(force: bool = False, verbose: bool = True) -> str:
    import sysconfig
    target = fast_module_path()
    header = os.path.join(HERE, "..", "include", "mia_hip.h")
    deps = [header, os.path.join(HERE, "_proto.py"), os.path.abspath(__file__)]
    if not force and os.path.exists(target) and all(os.path.getmtime(d) <= os.path.getmtime(target) for d in deps):
        return target
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    src = os.path.join(HERE, "build", "_mia_fast.c")
    with open(src, "w") as f:
        f.write(generate_fast_source())
    cmd = [os.environ.get("CC", "gcc"), "-O2", "-fPIC", "-shared", "-I" + sysconfig.get_paths()["include"], src, "-o", target]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return target


# ------------------------------------------------------------------------------------------------
# Autograd nodes in C++ (csrc/autograd.cpp): host code against torch's headers, linked to the library next to it.
# ------------------------------------------------------------------------------------------------
def autograd_module_path() -> str:
    import sysconfig
    return os.path.join(HERE, "_mia_autograd" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))


def build_autograd(force: bool = False, verbose: bool = True) -> str:
    import importlib.util
    import sysconfig
    target, src = autograd_module_path(), os.path.join(CSRC, "autograd.cpp")
    deps = [src, os.path.join(HERE, "..", "include", "mia_hip.h"), os.path.join(HERE, "_proto.py"), os.path.abspath(__file__)]
    spec = importlib.util.spec_from_file_location("mia_proto", os.path.join(HERE, "_proto.py"))
    proto = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(proto)
    import torch
    digest = proto.autograd_digest()
    if not force and os.path.exists(target) and all(os.path.getmtime(d) <= os.path.getmtime(target) for d in deps):
        with open(target, "rb") as f:       # another torch changes no file here, but the module is refused for it
            if digest.encode() + b"\0" in f.read():
                return target
    home = os.path.dirname(torch.__file__)
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-fPIC", "-shared", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f'-DMIA_HEADER_DIGEST="{digest}"',
           "-isystem", os.path.join(home, "include"), "-isystem", os.path.join(home, "include", "torch", "csrc", "api", "include"),
           "-isystem", os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"), "-isystem", sysconfig.get_paths()["include"],
           src, "-o", target, "-L" + os.path.join(home, "lib"), "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip", "-ltorch_python",
           "-L" + HERE, "-lmia_hip", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return target


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    build_fast(force="--force" in sys.argv)
    build_autograd(force="--force" in sys.argv)
    print(LIB)
