"""What the HIP runtime of this machine can do, asked without this library's
code (its symbols are reached through the library, so it is the runtime that
the library calls). Prints one JSON line {name: hip status, 0 = it can}.

    peer_import    importing a shareable allocation (a POSIX descriptor) that
                   another process exported
    host_register  registering host memory that already exists

Run as a program: it starts two processes of its own, so that the process that
asks keeps no device state and no error behind."""
import ctypes
import json
import os
import socket
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FD_TYPE = 1           # hipMemHandleTypePosixFileDescriptor


def runtime():
    sys.path.insert(0, ROOT)
    import torch.distributed  # noqa: F401  (the tests' workers load its runtime first)
    from xucg_amd import _lib
    return _lib.dev()


def take(hip, box, fd, by_value):
    """status of an import of fd: its number, or the address of an int that holds it"""
    box[0] = fd
    arg = fd if by_value else ctypes.addressof(box)
    return hip.hipMemImportFromShareableHandle(ctypes.byref(ctypes.c_void_p()), ctypes.c_void_p(arg), FD_TYPE)


def exporter(sock):
    hip, box, own, fd = runtime(), (ctypes.c_int * 4)(), ctypes.c_void_p(), ctypes.c_int(-1)
    # hipMemAllocationProp: pinned, descriptors wanted, on device 0, the rest 0
    prop = (ctypes.c_int * 16)(1, FD_TYPE, 1, 0)
    st = (hip.hipSetDevice(0) or
          hip.hipMemCreate(ctypes.byref(own), ctypes.c_size_t(2 << 20), prop, ctypes.c_ulonglong(0)) or
          hip.hipMemExportToShareableHandle(ctypes.byref(fd), own, FD_TYPE, ctypes.c_ulonglong(0)))
    # the address first: a runtime that reads it must never get a number
    by_value = st == 0 and take(hip, box, fd.value, False) != 0
    st = st or (take(hip, box, fd.value, True) if by_value else 0)
    socket.send_fds(sock, [json.dumps([st, by_value]).encode()], [] if st else [fd.value])
    sock.recv(1)
    return {}


def importer(sock):
    hip = runtime()
    buf = (ctypes.c_char * (1 << 20))()
    msg, fds, _, _ = socket.recv_fds(sock, 64, 1)
    st, by_value = json.loads(msg)
    answers = {}
    if hip.hipSetDevice(0) == 0:          # without a device nothing is known
        answers["host_register"] = hip.hipHostRegister(buf, ctypes.c_size_t(len(buf)), ctypes.c_uint(0))
        if answers["host_register"] == 0:
            hip.hipHostUnregister(buf)
        if st == 0:                       # the exporter has it, and could import it itself
            answers["peer_import"] = take(hip, (ctypes.c_int * 4)(), fds[0], by_value)
    sock.send(b"y")
    return answers


def main():
    if len(sys.argv) > 1:
        out = {"export": exporter, "import": importer}[sys.argv[1]](socket.socket(fileno=int(sys.argv[2])))
        if out:
            print(json.dumps(out), flush=True)
        return 0
    a, b = socket.socketpair()
    ps = [subprocess.Popen([sys.executable, os.path.abspath(__file__), side, str(s.fileno())],
                           pass_fds=[s.fileno()]) for side, s in (("export", a), ("import", b))]
    a.close()
    b.close()
    return max(abs(p.wait(timeout=100)) for p in ps)


if __name__ == "__main__":
    sys.exit(main())
