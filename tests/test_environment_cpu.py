"""A call's result is its arguments' alone: the library reads no environment variable in a call."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# getenv as it is, with a note of every name asked for
SPY = r'''
#define _GNU_SOURCE
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
extern char **environ;
static int noting;
void note_names(int on) { noting = on; }
char *getenv(const char *name) {
    if (noting) fprintf(stderr, "asked for %s\n", name);
    size_t n = strlen(name);
    for (char **e = environ; e && *e; ++e)
        if (!strncmp(*e, name, n) && (*e)[n] == '=') return *e + n + 1;
    return NULL;
}
char *secure_getenv(const char *name) { return getenv(name); }
'''

# operands that are never read: the process sees no device
CALLS = r'''
import ctypes, sys
sys.path.insert(0, sys.argv[1])
from hidet_b200 import ffi
at = 4096
calls = [lambda: ffi.func('b200q_quantize_tokens')(at, 64, None, 1e-6, at, at, 2, 64, ffi.F16, None),
         lambda: ffi.func('b200q_route_tokens')(at, 64, at, at, at, 2, 64, 8, 2, 0, ffi.F16, ffi.F16, None),
         lambda: ffi.func('b200q_mixture_of_experts')(at, 64, at, at, at, at, at, at, None, 0, at, 2, 64, 32, 8, 2, ffi.F16, ffi.F16, at, 1 << 30, None),
         lambda: ffi.func('b200q_symmetric_quantize')(at, at, at, 64, 64, ffi.F16, ffi.I8, 0, None),
         lambda: ffi.func('b200q_qlinear_f16_i8')(at, at, at, at, 2, 64, 64, 0, at, 1 << 30, None)]
for m, n, k in ((2, 64, 64), (2000, 4096, 4096), (3, 63, 61)):
    for layout in (0, 1):
        calls.append(lambda m=m, n=n, k=k, layout=layout: ffi.func('b200q_qlinear_i8_i8')(at, at, at, at, at, m, n, k, layout, ffi.F16, ffi.F16, None, None))
note = ctypes.CDLL(None).note_names
for on in (0, 1):   # what is read once for the process, when it first looks for a device, is read by then
    note(on)
    for call in calls:
        try:
            call()
        except ffi.BackendException:
            pass
note(0)
print('called', len(calls))
'''


@pytest.mark.skipif(shutil.which('gcc') is None, reason='no C compiler')
def test_calls_read_no_environment_variable(tmp_path):
    source, spy = str(tmp_path / 'spy.c'), str(tmp_path / 'spy.so')
    open(source, 'w').write(SPY)
    subprocess.check_call(['gcc', '-O1', '-fPIC', '-shared', source, '-o', spy])
    done = subprocess.run([sys.executable, '-c', CALLS, ROOT], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=600,
                          env=dict(os.environ, LD_PRELOAD=spy, CUDA_VISIBLE_DEVICES=''))
    assert done.returncode == 0 and done.stdout.startswith('called'), done.stderr
    # CUDA's runtime, which looks for a driver again with every call where there is none, has names of its own
    asked = {line.split()[-1] for line in done.stderr.splitlines() if line.startswith('asked for ')}
    assert not {name for name in asked if not name.startswith(('CUDA', 'NV', 'LD_', 'GLIBC'))}, asked
