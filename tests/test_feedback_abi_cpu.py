"""The feedback operators' C entries refuse what their kernels cannot work on.  Never dereferenced: every call is refused before its launch."""
import ctypes

import pytest


@pytest.mark.parametrize('off', [1, 4])
def test_misaligned_partials_and_workspaces(off):
    from learning_embeddings_amd import _lib
    lib, p, q = _lib.lib, ctypes.c_void_p(256), ctypes.c_void_p(256 + off)
    sizes = ctypes.cast((ctypes.c_int32 * 2)(2, 3), ctypes.c_void_p)
    w = lib.lec_path_workspace_bytes()
    for call in (lambda: lib.lec_path_logp_fwd(p, 0, 5, 1, 5, sizes, 2, p, 1, p, q, None), lambda: lib.lec_path_logp_bwd(p, 0, 5, 1, 5, sizes, 2, p, 1, q, p, None, None, p, 5, None),
                 lambda: lib.lec_preference_loss_fwd(p, 0, 5, 1, 1, 5, sizes, 2, p, p, 0.1, 0.0, p, p, p, q, p, w, None),
                 lambda: lib.lec_preference_loss_fwd(p, 0, 5, 1, 1, 5, sizes, 2, p, p, 0.1, 0.0, p, p, p, p, q, w, None),
                 lambda: lib.lec_policy_loss_fwd(p, 0, 5, 1, 5, sizes, 2, p, 1, p, None, None, 0.2, 0.2, 0.0, 0, p, p, p, p, q, p, w, None),
                 lambda: lib.lec_policy_loss_fwd(p, 0, 5, 1, 5, sizes, 2, p, 1, p, None, None, 0.2, 0.2, 0.0, 0, p, p, p, p, p, q, w, None)):
        assert call() == _lib.E_ARG and b'aligned' in lib.lec_last_error()
