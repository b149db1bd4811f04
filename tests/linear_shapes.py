"""Shapes that reach every kernel of the 16-bit and 4-bit products, unsplit and split along K wherever their plans split them,
and products in parts along rows and columns. Ragged: rows, columns and K end inside a tile, a stage and a piece of 16 bytes."""

KERNELS = ["tile 256x256", "tile 256x128", "tile 128x128", "int4 256x256", "int4 128x256", "few 16 1/16/1", "few 16 1/8/2",
           "few 16 2/8/1", "few 16 2/4/2", "few 16 2/16/1", "few 32 1/4/4", "few 32 2/4/4", "few 32 2/4/2", "few 32 4/4/2",
           "few 64 2/4/2"]

# Of a kind of product: (rows, outputs, K) -> its launches, each a kernel and whether K is split.
PRODUCT = {
    (1, 33, 40): [("tile 128x128", False)],
    (3, 35, 1037): [("tile 128x128", True)],
    (1301, 10301, 523): [("tile 256x256", False)],
    (203, 20997, 4101): [("tile 256x128", False)],
    (701, 4203, 16390): [("tile 256x128", True)],
    (1003, 5203, 8197): [("tile 256x256", True)],
    (1001, 16501, 1035): [("tile 256x256", False), ("tile 128x128", True)],
    (1301, 4201, 16391): [("tile 256x256", True), ("tile 128x128", True)],
}
GATED = {
    (1, 33, 40): [("few 16 2/8/1", False)],
    (3, 35, 4104): [("few 16 2/8/1", True)],
    (3, 4203, 8200): [("few 16 2/4/2", False)],
    (5, 45, 8200): [("few 16 2/4/2", True)],
    (19, 10301, 72): [("few 32 4/4/2", False)],
    (17, 33, 136): [("few 32 2/4/2", False)],
    (23, 45, 2056): [("few 32 2/4/2", True)],
    (39, 33, 520): [("few 64 2/4/2", False)],
    (61, 45, 2056): [("few 64 2/4/2", True)],
    (65, 33, 40): [("tile 128x128", False)],
    (67, 45, 1032): [("tile 128x128", True)],
    (1301, 5205, 520): [("tile 256x256", False)],
    (501, 5205, 8200): [("tile 256x256", True)],
    (701, 3101, 4104): [("tile 256x128", False)],
    (703, 2101, 16392): [("tile 256x128", True)],
    (1303, 3101, 520): [("tile 128x128", False)],
    (1301, 2101, 16392): [("tile 256x256", True), ("few 32 2/4/2", True)],
    (1001, 8301, 1032): [("tile 256x256", False), ("tile 128x128", True)],
}
INT4 = {
    (1, 33, 39): [("few 16 1/16/1", False)],
    (3, 35, 16389): [("few 16 1/16/1", True)],
    (9, 4203, 71): [("few 16 1/8/2", False)],
    (11, 8301, 133): [("few 16 2/8/1", False)],
    (17, 33, 135): [("few 32 1/4/4", False)],
    (23, 45, 2055): [("few 32 1/4/4", True)],
    (39, 33, 519): [("few 64 2/4/2", False)],
    (61, 45, 2055): [("few 64 2/4/2", True)],
    (65, 33, 39): [("int4 128x256", False)],
    (67, 45, 1031): [("int4 128x256", True)],
    (70, 45, 4103): [("few 64 2/4/2", True), ("few 16 1/16/1", False)],
    (701, 21005, 519): [("int4 256x256", False)],
    (703, 10301, 4103): [("int4 256x256", True)],
    (1001, 16501, 1031): [("int4 256x256", False), ("int4 128x256", True)],
    (1025, 5203, 4103): [("int4 128x256", True), ("few 16 1/8/2", False)],
}
INT4_GATED = {
    (1, 33, 39): [("few 16 2/8/1", False)],
    (3, 35, 8190): [("few 16 2/8/1", True)],
    (3, 35, 8197): [("few 16 2/16/1", False)],
    (5, 35, 16389): [("few 16 2/16/1", True)],
    (9, 8301, 71): [("few 16 2/4/2", False)],
    (19, 10301, 71): [("few 32 2/4/4", False)],
    (17, 33, 135): [("few 32 2/4/2", False)],
    (23, 45, 2055): [("few 32 2/4/2", True)],
    (39, 33, 519): [("few 64 2/4/2", False)],
    (61, 45, 2055): [("few 64 2/4/2", True)],
    (65, 33, 39): [("int4 128x256", False)],
    (67, 45, 1031): [("int4 128x256", True)],
    (99, 45, 4103): [("few 64 2/4/2", True), ("few 64 2/4/2", True)],
    (701, 5205, 4103): [("int4 256x256", True)],
    (1001, 8301, 1031): [("int4 256x256", False), ("int4 128x256", True)],
    (1301, 3101, 4103): [("int4 256x256", True), ("few 32 2/4/2", True)],
}
# Which of the kernels have no K split in any plan.
NEVER_SPLIT = {"few 16 1/8/2", "few 32 4/4/2", "few 32 2/4/4"}
