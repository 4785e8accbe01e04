"""The launchers behind include/ie_kv8.h's attention (csrc/kv8.h), which the engine calls by themselves."""
import ctypes

I, P = ctypes.c_int, ctypes.c_void_p


class CacheArgs(ctypes.Structure):  # Kv8Cache
    _fields_ = [(n, P) for n in ("k", "v", "ks", "vs", "table")] + [(n, I) for n in ("nbps", "H", "d", "bs_log2")]


class AttnArgs(ctypes.Structure):  # Kv8Attn
    _fields_ = [("B", I), ("P", I), ("H_q", I), ("Q", P), ("q_ld", I), ("c", CacheArgs), ("lens", P), ("max_ctx", I),
                ("start", I), ("O", P), ("ws", P), ("splits", I), ("K", P), ("V", P), ("kv_ld", I), ("positions", P),
                ("undo_at", P), ("undo_scale", P), ("undo_codes", P)]


NAMES = {"decode": "_ZN2ie22launch_decode_attn_kv8ERKNS_7Kv8AttnEP12ihipStream_t",
         "prefill": "_ZN2ie23launch_prefill_attn_kv8ERKNS_7Kv8AttnEP12ihipStream_t"}


def launch(ie, which, args, stream=None):
    """The launcher's status."""
    ie.load()
    return ctypes.CDLL(ie.LIB_PATH)[NAMES[which]](ctypes.byref(args), P(stream))
