"""A call of each form that the attention over 4-bit caches has (csrc/attn4_plan.hpp): (n_head, n_head_kv, D, T, n_kv) and the
columns of the matrix instruction a row and the groups of rows a workgroup that it is cut into."""
FORMS = {
    (14, 2, 64, 1, 200): (2, 1), (14, 2, 64, 33, 900): (2, 1), (32, 8, 64, 100, 700): (1, 1), (32, 8, 64, 600, 333): (1, 2),
    (32, 8, 128, 1, 2000): (4, 1), (8, 1, 128, 20, 700): (2, 1), (32, 8, 128, 80, 1000): (1, 1), (32, 8, 128, 520, 300): (1, 2),
    (8, 4, 256, 1, 900): (4, 1), (8, 1, 256, 10, 600): (2, 1), (8, 4, 256, 300, 300): (1, 1),
    (4, 2, 512, 3, 500): (4, 1), (8, 1, 512, 20, 400): (2, 1), (16, 1, 512, 5, 300): (1, 1),
}
