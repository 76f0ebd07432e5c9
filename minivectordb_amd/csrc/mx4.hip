// mx4.hip -- kernels of the microscaled 4-bit operators (format and entry points: mx4.hpp)
#include "mx4.hpp"

#include "mx4_rows.hip.hpp"
#include "mx4_product.hip.hpp"
#include "mx4_scan.hip.hpp"
