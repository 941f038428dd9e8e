"""Plain statements of the calls for drafted tokens, forks and log probabilities, to put in the kernels' place on the CPU."""
from __future__ import annotations

import torch

import kernel_refs
import plain_drafts as plain


def qk_norm_rope_store(*args, places=None, **more):
    """With ``places`` a row turns by its position and is stored at its place: the plain statement once for the queries, once (with tables
    whose row p holds the angles of the row stored at p) for the rest."""
    if places is None:
        return kernel_refs.qk_norm_rope_store(*args, **more)
    args = list(args)
    cos, sin, positions, row_request = args[8], args[9], args[11], args[12]
    qkv, q_out = args[0], args[16]
    for r in range(qkv.shape[0]):
        one = list(args)
        p, at = int(positions[r]), int(places[r])
        if args[10]:
            one[8], one[9] = cos[p][None].expand(at + 1, -1), sin[p][None].expand(at + 1, -1)
        one[0], one[11], one[12], one[16] = qkv[r:r + 1], places[r:r + 1], row_request[r:r + 1], q_out[r:r + 1]
        kernel_refs.qk_norm_rope_store(*one, **more)


def paged_attention_tree(q, k_pages, v_pages, block_table, q_start, context, positions, seen, scale, window, out, max_tree, max_kv_len):
    assert max_tree >= int((q_start[1:] - q_start[:-1]).max()) and max_kv_len >= int((context + q_start[1:] - q_start[:-1]).max())
    o, _ = plain.tree_attention(q, k_pages, v_pages, block_table, q_start, context, positions, seen, scale, window or 0)
    out.copy_(o.flatten(1).to(out.dtype))


def _planes(pages, axis):
    return pages.view((-1,) + pages.shape[axis:])


def copy_pages(pages, axis, source, target):
    p = _planes(pages, axis)
    for a, b in zip(source.tolist(), target.tolist()):
        p[:, b] = p[:, a]


def keep_tokens(pages, axis, block_table, context, kept, n_kept):
    p = _planes(pages, axis)
    size = p.shape[3]
    for r, n in enumerate(n_kept.tolist()):
        for i in range(n):
            a, b = int(context[r]) + int(kept[r, i]), int(context[r]) + i
            pa, pb = int(block_table[r, a // size]), int(block_table[r, b // size])
            if pa >= 0 and pb >= 0:
                p[:, pb, :, b % size] = p[:, pa, :, a % size].clone()


def token_log_probs(logits, tokens, log_probs, entropy=None, top_ids=None, top_log_probs=None):
    lp, h, ids, best = plain.log_probs(logits, tokens, 0 if top_ids is None else top_ids.shape[1])
    log_probs.copy_(lp)
    if entropy is not None:
        entropy.copy_(h)
    if top_ids is not None:
        top_ids.copy_(ids)
        top_log_probs.copy_(best)


def install(monkeypatch):
    import inferrs_b200.kernels as K

    kernel_refs.install(monkeypatch)
    for name in ("qk_norm_rope_store", "paged_attention_tree", "copy_pages", "keep_tokens", "token_log_probs"):
        monkeypatch.setattr(K, name, globals()[name])
