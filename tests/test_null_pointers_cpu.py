"""Entry points of the embedding, the token loss and the 8-bit activations answer null pointers with an error code before they touch a device."""
import ctypes as C

from sneppx_alg_b200 import _build
from sneppx_alg_b200.ops._lib import SxVocabLossArgs


def _calls(lib, name, types, args, pointers):
    """The entry point's answer with each of its needed pointers null in turn."""
    fn = getattr(lib, name)
    fn.argtypes, fn.restype = types, C.c_int
    for k in pointers:
        yield name, k, fn(*[0 if i == k else a for i, a in enumerate(args)])


def test_null_pointers_are_refused():
    lib = C.CDLL(str(_build.build_cuda()))                 # a handle of its own: argument types are set here
    p, i, l, f = C.c_void_p, C.c_int, C.c_longlong, C.c_float
    at = 1 << 12                                           # aligned, and never read
    checks = [
        _calls(lib, "sx_embed_fwd", [p, i, p, l, p, l, i, l, f, i, l, p, p, p], [at, 1, at, 8, at, 4, 8, 5, 1.0, 0, -1, 0, at, 0], (0, 2, 4)),
        _calls(lib, "sx_embed_bwd", [p, i, p, p, l, l, i, l, l, f, i, i, i, p, p, l, p, p],
               [at, 1, at, at, 8, 4, 8, 5, -1, 1.0, 0, 0, 0, 0, at, 1 << 30, at, 0], (0, 2, 3, 14)),
        _calls(lib, "sx_vocab_loss_fwd", [p, l, p, l, p, l, l, i, l, f, p, p, p, p, p, p], [at, 8, at, 8, at, 4, 5, 8, -100, 0.0, at, at, at, at, at, 0],
               (0, 2, 4, 10, 11, 12, 13)),
        _calls(lib, "sx_pack8", [p, p, p, l, i, l, i, p], [at, at, at, 4, 32, 32, 0, 0], (0, 1, 2)),
        _calls(lib, "sx_unpack8", [p, p, p, l, i, l, i, p], [at, at, at, 4, 32, 32, 0, 0], (0, 1, 2)),
        _calls(lib, "sx_glu8_fwd", [p, p, p, p, l, i, l, i, i, p], [at, at, at, at, 4, 32, 64, 0, 0, 0], (0, 1, 2, 3)),
        _calls(lib, "sx_glu8_bwd", [p, p, p, p, l, i, i, i, p], [at, at, at, at, 4, 32, 0, 0, 0], (0, 1, 2, 3)),
    ]
    for name, k, rc in (c for group in checks for c in group):
        assert rc == -1, (name, k, rc)
    lib.sx_vocab_loss_bwd.argtypes, lib.sx_vocab_loss_bwd.restype = [p, p], C.c_int
    for missing in ("h", "w", "target", "lse", "nll", "work"):
        a = SxVocabLossArgs(h=at, w=at, ldh=8, ldw=8, target=at, lse=at, nll=at, dh=at, dw=at, lddw=8, T=4, V=5, ignore_index=-100, work=at,
                            work_bytes=1 << 40, d=8)
        setattr(a, missing, None)
        assert lib.sx_vocab_loss_bwd(C.addressof(a), None) == -1, missing
