"""Whether a call over shared prefixes took them up, by what it left in its workspace."""
import torch


def shared_workspace(q, keys, table):
    from moss_tts._runtime import paged

    return paged.shared_decode_workspace(q, keys, table).fill_(float("nan"))


def prefix_taken(ws, q, keys):
    """The partial results of prefixes lie behind those of the sequences' own rows: 4 for a workgroup and one a sequence."""
    (b, qh, d), kh = q.shape, keys.shape[1]
    own = (4 * max(512 // kh, 2) + b) * qh * d
    return bool(torch.isfinite(ws[own:own + b * qh * d]).any())
