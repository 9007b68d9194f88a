// The index arithmetic of attention over shared prefixes, compiled for the host out of the kernels' own header, beside what paged_host.cpp has.
#include "paged_host.cpp"

extern "C" {

// 1: a group whose numbers can be, and its first row, rows, first token, tokens and shared tokens; *err as the kernels would leave it
int host_group_span(const uint32_t* starts, const uint32_t* lens, int64_t rows, int64_t cols, int lg, int64_t M, const uint32_t* groups, const uint32_t* shared, int64_t n,
                    int64_t most, int64_t group, int64_t* out, int32_t* err) {
  PagedRows p = {starts, lens, nullptr, rows, cols, M, 0, lg, err};
  PagedGroups g = {groups, shared, n, most};
  return group_span(p, g, group, out, out + 1, out + 2, out + 3, out + 4);
}
int64_t host_position_of(const uint32_t* starts, const uint32_t* lens, int64_t rows, int64_t row0, int64_t count, int64_t token) {
  PagedRows p = {starts, lens, nullptr, rows, 0, 0, 0, 0, nullptr};
  return position_of(p, row0, count, token);
}

}
