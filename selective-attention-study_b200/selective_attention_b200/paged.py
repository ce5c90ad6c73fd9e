"""A paged cache for Selective Attention: many requests of different lengths, answered together.

The dense cache of ``SelectiveAttentionSlot`` holds sequences of one length; here every row (a request, or a beam of one) owns
pages of ``page_size`` tokens.  All of it is plain tensors in plain dicts:

    tables   shared by every layer of a model: "block_tables" (rows, max_pages) int32, -1 where a row has no page; "lengths"
             (rows,); "free_pages" (num_pages,), of which the first "free_count" are free; "page_refs" (num_pages,), the rows that
             hold a page; "page_size"; "heads"
    cache    of one layer: "k", "v" (num_pages, H, page_size, D) bf16; "selected" (rows, G, max_pages * page_size) fp32, the
             selection that every key has received (G = 1: head 0 selects for all; G = H: every head for itself)
    step     what a step of the server needs, made once for all layers by ``append_tokens``
    moves    what ``reorder_rows`` has decided, carried out in every layer by ``move_rows``

A step: ``append_tokens`` hands out pages for the new tokens of every row (a prompt, a further chunk of one, or a single token),
``paged_attention`` of every layer stores their keys and values and attends to them.  The numbers of tokens stay on the GPU: no
call waits for it, and a step can be captured in a graph.  There is no counterpart in the reference, whose cache is one contiguous
tensor per layer (``mixers.py:105-130``).  CUDA tensors and the built library only.
"""

from __future__ import annotations

import torch

from . import _lib, kernels

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_ROWS = 4096


def begin_tables(rows: int, num_pages: int, page_size: int, max_pages: int, heads: int, device="cuda") -> dict:
    """Tables of ``rows`` empty rows over a pool of ``num_pages`` free pages; a row has room for ``max_pages`` of them.  ``heads``
    are those of the layers that will share the tables (the plan of a step divides its work by them)."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}; got {page_size}")
    if not 1 <= rows <= MAX_ROWS or num_pages < 1 or max_pages < 1 or not 1 <= heads <= 256:
        raise ValueError(f"1 to {MAX_ROWS} rows, at least one page, 1 to 256 heads; got {rows}, {num_pages}, {max_pages}, {heads}")

    def ints(*shape, fill):
        return torch.full(shape, fill, dtype=torch.int32, device=device)

    return {"block_tables": ints(rows, max_pages, fill=-1), "lengths": ints(rows, fill=0),
            "free_pages": torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device),
            "free_count": ints(1, fill=num_pages), "page_refs": ints(num_pages, fill=0), "page_size": int(page_size), "heads": int(heads)}


def begin_pages(tables: dict, head_dim: int, per_head: bool = False) -> dict:
    """The pools and histories of one layer."""
    rows, max_pages = tables["block_tables"].shape
    heads, page, device = tables["heads"], tables["page_size"], tables["block_tables"].device
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128 in a paged cache; got {head_dim}")
    pool = (tables["page_refs"].numel(), heads, page, head_dim)
    return {"k": torch.zeros(pool, dtype=torch.bfloat16, device=device), "v": torch.zeros(pool, dtype=torch.bfloat16, device=device),
            "selected": torch.zeros(rows, heads if per_head else 1, max_pages * page, dtype=torch.float32, device=device)}


def append_tokens(tables: dict, counts: torch.Tensor, total: int, max_length: int | None = None, max_count: int | None = None) -> dict:
    """Row r gets ``counts[r]`` (int32, on the GPU) new tokens; the tables have their pages afterwards.  ``total``: how many tokens the
    step has; q, k, v of its attention hold them row after row.

    ``max_length`` and ``max_count`` are bounds that the host knows: no row is longer after the step, no row gets more tokens.  They
    set scratch and launches (a step with a max_count of up to 8 is a decode step: one launch a layer); by default they are what
    the tables allow.

    Returns "query_start" (rows + 1,) int32, where each row's tokens start (cut at ``total``); "cached" (rows,) int32, the tokens
    before the step; "slots" (total,) int64, page * page_size + offset of every token.  A row that does not fit -- its table, the
    bounds, ``total``, or the pool, and then no later row that needs a page fits either -- is left as it was: "cached" and its
    slots are -1, its outputs zeros.  A token behind the last row has slot -1 too."""
    native = _lib.native()
    most = tables["block_tables"].shape[1] * tables["page_size"]
    max_length = most if max_length is None else int(max_length)
    made = native.append_tokens(tables, counts, int(total), max_length, most if max_count is None else int(max_count))
    return {"query_start": made[0], "cached": made[1], "slots": made[2], "_plan": made[3]}


def paged_attention(cache: dict, tables: dict, step: dict, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, exempt: int = 1) -> torch.Tensor:
    """Selective Attention of the step's tokens: q, k, v (total, H, D), any token and head strides.  Stores k and v in the pages, returns
    (total, H, D) bf16 -- row r's tokens get what ``selective_attention`` over all tokens of the row gives its last ones -- and
    moves ``cache["selected"]`` on.  Tokens without a slot get zeros.  The cache is bf16 and so are its products: q, k, v in fp16 or
    fp32 are rounded to it first (2^-8, where a dense cache keeps their type).

    One call per layer and step; calls of one step on one stream share its plan.  Nothing behind a row's last token is read
    into a result or written."""
    return _lib.native().paged_attention(tables, step["_plan"], cache["k"], cache["v"], cache["selected"], q, k, v,
                                         kernels._check_exempt(exempt))


def reorder_rows(tables: dict, parents: torch.Tensor) -> dict:
    """Row r becomes a copy of row ``parents[r]`` (int32, on the GPU; outside [0, rows): an empty row, so -1 gives a row's pages back).
    Beams do this after every selection, a prompt that is answered several times does it once.

    Full pages are shared between the copies.  The page that is still being filled stays with the lowest row that has the
    parent; the others get a page of their own, and ``move_rows`` copies its tokens in every layer: "copies" (rows, 2) int32
    holds source and target, or -1, -1.  Pages that nobody holds any more go back first, lowest first.  A row that needs a page
    when there is none becomes empty: "lost" (1,) int32 is how many did, and their "lengths" are 0.  What they were is gone, so a
    search that must not lose a beam keeps a free page for every row."""
    copies, work, lost = _lib.native().reorder_rows(tables, parents)
    return {"copies": copies, "lost": lost, "tables": tables, "_work": work}


def move_rows(cache: dict, moves: dict) -> None:
    """Carries out ``moves`` in one layer: the tokens of the copied pages, and the histories of the rows."""
    _lib.native().move_rows(moves["tables"], moves["copies"], moves["_work"], cache["k"], cache["v"], cache["selected"])
