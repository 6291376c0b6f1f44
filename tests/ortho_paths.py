"""Lists of matrices that take every path of the orthogonalisation's products: which tile,
whole or in parts or with the last round alone in parts, in one word or two, wide or tall
(tests/test_ortho_plan.py checks that they do).  (precision, [(rows, cols, how many)])"""

LISTS = [
    ("fast", [(231, 768, 1), (55, 16, 4), (64, 64, 24)]),
    ("fp32", [(21, 86, 1), (701, 259, 1)]),
    ("fast", [(192, 1713, 1), (1052, 718, 1)]),
    ("fast", [(1344, 143, 24), (145, 347, 8)]),
    ("fast", [(571, 33, 1)]),
    ("fp32", [(275, 5422, 4), (384, 19, 1)]),
    ("fast", [(31, 62, 2), (256, 41, 1), (1856, 930, 24)]),
    ("fp32", [(704, 668, 24), (568, 1717, 1), (161, 34, 4)]),
    ("fp32", [(1940, 2005, 2), (1664, 48, 1)]),
    ("fp32", [(47, 51, 2), (2240, 1808, 1)]),
    ("fast", [(2143, 1984, 4), (24, 872, 4), (210, 2082, 1)]),
    ("fast", [(142, 2080, 1), (2176, 1536, 24), (640, 29, 8)]),
    ("fast", [(576, 1198, 2), (666, 757, 24), (181, 724, 8)]),
    ("fp32", [(26, 920, 8), (29, 28, 4), (1472, 1472, 24)]),
    ("fast", [(1344, 74, 2), (3064, 3260, 1)]),
    ("fast", [(3685, 3016, 1)]),
]


def matrices(shapes):
    """(rows, cols) of every matrix"""
    return [(m, n) for m, n, many in shapes for _ in range(many)]
