"""Float64 restatement of the token embedding and its gradient (no reference code).

  out[i] = scale * table[ids[i]], 0 where ids[i] is outside [0, V)
  dtable[v] = scale * sum of dout[i] over ids[i] = v
"""

import numpy as np

__all__ = ["embedding", "embedding_bwd"]


def embedding(table, ids, scale=1.0):
    """[..., C] float64 for table [V,C] and ids of any shape."""
    table, ids = np.asarray(table, np.float64), np.asarray(ids)
    out = np.zeros(ids.shape + (table.shape[1],))
    there = (ids >= 0) & (ids < table.shape[0])
    out[there] = scale * table[ids[there]]
    return out


def embedding_bwd(dout, ids, rows, scale=1.0):
    """[rows,C] float64 for dout [..., C]."""
    dout, ids = np.asarray(dout, np.float64), np.asarray(ids)
    dtable = np.zeros((rows, dout.shape[-1]))
    there = (ids >= 0) & (ids < rows)
    np.add.at(dtable, ids[there], dout[there])
    return scale * dtable
