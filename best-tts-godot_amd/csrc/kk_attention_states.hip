#include "kk_attention.h"
namespace kk {
bool few_dense_try(const QueryArgs&, const DenseArgs&, int, int*) { return false; }
}
